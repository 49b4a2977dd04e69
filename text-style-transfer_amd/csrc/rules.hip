// Rules on the logits of a step: penalties for repeated tokens, biases, grammar masks; and the step of a grammar's states.
#include "tst_common.h"

namespace {

constexpr int CHUNK_L = 8192, NT_L = 512;   // columns and threads of a workgroup where there are many rows
constexpr int LIST = 2048;                  // columns that the list holds
constexpr uint32_t SEEN = 0x80000000u;   // counter bit: the token is in the prompt

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));   // four floats at any float's address
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }
// 16 bytes of logits
template <typename T>
struct Piece {
    uint4 u;
    __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void values(float (&x)[4]) const {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    }
    __device__ __forceinline__ void values(float (&x)[8]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
};
__device__ __forceinline__ void store16(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void store16(__bf16* p, const float (&x)[8]) {
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (__bf16)x[e];
    *reinterpret_cast<bf16x8*>(p) = v;
}

// One workgroup per row and chunk of CHUNK columns, HBM-bound: the logits are read and written once, the row's tokens once per chunk out of
// the caches.
//   1. The row's tokens are counted in LDS, one 32-bit counter per column (integer atomics: the order does not matter); whoever finds
//      a counter at 0 puts the column on a list.
//   2. The listed columns' logits are penalised and left in place of their counters, as the complement of their bits (0 = no such
//      token): a few divisions per row with all lanes at work, instead of a branch per column in the stream.
//   3. The chunk streams through, 16 bytes per lane: penalised value or logit, bias, mask.
// Chunks begin where the row's addresses are 16-byte aligned, whatever the row's own alignment (`shift` columns before it); a row is only
// handled element by element where logits and out are aligned differently.  In place (`out` is `logits`), pieces that no rule changes
// are neither read nor written.
// 2048 rows of 32000 bf16 logits with bias, masks and 1300 tokens each: 69.7 us, 3.8 TB/s; without rules 50 (a copy: 50), the bias 7, the
// tokens 9 to 13 of it.  The list is short so that four workgroups share a CU (with room for every column, three: 72.5).  Measured beside
// it: the bias requested with the logits 80 us, after the counting 74, chunks of 4096 with 256 threads 78, each workgroup taking rows in
// turn with the next one's inputs under way 128, the simple kernel, a branch per column, 322.
template <typename T, int CHUNK, int NT>
__global__ __launch_bounds__(NT) void adjust_logits_kernel(const T* logits, int64_t ld, int V, tst_logit_rules a, T* out, int64_t ldo) {
    __shared__ __attribute__((aligned(16))) uint32_t count[CHUNK];
    __shared__ uint16_t list[LIST];
    __shared__ int listed;
    constexpr int E = 16 / (int)sizeof(T);
    const int t = threadIdx.x;
    const int64_t r = blockIdx.y;
    const T* row_in = logits + r * ld;
    T* row_out = out + r * ldo;
    const int shift = (int)((reinterpret_cast<uintptr_t>(row_in) & 15u) / sizeof(T));
    const bool vec = ((reinterpret_cast<uintptr_t>(row_in) ^ reinterpret_cast<uintptr_t>(row_out)) & 15u) == 0u;
    const int v0 = (int)blockIdx.x * CHUNK - shift;                  // column of count[0]; below 0 in the first chunk of an unaligned row
    if (v0 >= V) return;
    const int64_t s = a.sent != nullptr ? a.sent[r] : r;
    int p_lo = 0, p_hi = 0, n_hist = 0;
    float rp = 1.0f, fp = 0.0f, pp = 0.0f;
    if (a.params != nullptr && s >= 0 && s < a.n_sent) {
        rp = a.params[3 * s]; fp = a.params[3 * s + 1]; pp = a.params[3 * s + 2];
        if (a.prompt != nullptr) {
            p_lo = max(a.prompt_cu[s], 0);
            p_hi = min(a.prompt_cu[s + 1], (int)a.n_prompt);
        }
        if (a.hist != nullptr) n_hist = a.hist_len != nullptr ? min(a.hist_len[r], (int)a.n_hist) : (int)a.n_hist;
    }
    const bool penal = p_hi > p_lo || n_hist > 0;
    const int64_t br = a.bias == nullptr ? -1 : (a.bias_row != nullptr ? a.bias_row[r] : 0);
    const int64_t mr = a.mask == nullptr ? -1 : (a.mask_row != nullptr ? a.mask_row[r] : 0);
    const float* bias = br >= 0 && br < a.n_bias ? a.bias + br * a.ld_bias : nullptr;
    const uint32_t* mask = mr >= 0 && mr < a.n_masks ? a.mask + mr * a.ld_mask : nullptr;
    const int words = (V + 31) >> 5;
    // the chunk's logits and mask bits are requested before the tokens are counted, unless most of them will not be needed
    constexpr int PER = CHUNK / E / NT;
    const bool ahead = out != logits || bias != nullptr;
    Piece<T> x[PER];
    uint64_t bits[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int c0 = v0 + (t + NT * j) * E;
        const bool whole = vec && c0 >= 0 && c0 + E <= V;
        if (whole && ahead) x[j].load(row_in + c0);
        bits[j] = ~0ull;
        if (whole && mask != nullptr) {
            const int w = c0 >> 5;
            bits[j] = mask[w];
            if ((c0 & 31) + E > 32 && w + 1 < words) bits[j] |= (uint64_t)mask[w + 1] << 32;
        }
    }
    if (penal) {
        const int32_t* hist = a.hist + r * a.ld_hist;
        int vp[4], vh[4];                                            // the first tokens, requested as early
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            vp[u] = p_lo + t + NT * u < p_hi ? a.prompt[p_lo + t + NT * u] : -1;
            vh[u] = t + NT * u < n_hist ? hist[t + NT * u] : -1;
        }
        for (int i = t; i < CHUNK / 4; i += NT) reinterpret_cast<uint4*>(count)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (t == 0) listed = 0;
        __syncthreads();
        const int lo = max(v0, 0), n = min(v0 + CHUNK, V) - lo;
        auto note = [&](int v, bool prompt) {
            if ((uint32_t)(v - lo) >= (uint32_t)n) return;
            const uint32_t old = prompt ? atomicOr(&count[v - v0], SEEN) : atomicAdd(&count[v - v0], 1u);
            if (old == 0u) {
                const int at = atomicAdd(&listed, 1);
                if (at < LIST) list[at] = (uint16_t)(v - v0);
            }
        };
#pragma unroll
        for (int u = 0; u < 4; ++u) note(vp[u], true);
#pragma unroll
        for (int u = 0; u < 4; ++u) note(vh[u], false);
        for (int64_t at = (int64_t)p_lo + t + 4 * NT; at < p_hi; at += 4 * NT) {
#pragma unroll
            for (int u = 0; u < 4; ++u) vp[u] = at + NT * u < p_hi ? a.prompt[at + NT * u] : -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) note(vp[u], true);
        }
        for (int64_t at = t + 4 * NT; at < n_hist; at += 4 * NT) {
#pragma unroll
            for (int u = 0; u < 4; ++u) vh[u] = at + NT * u < n_hist ? hist[at + NT * u] : -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) note(vh[u], false);
        }
        __syncthreads();
        const bool all = listed > LIST;                              // more than the list holds: look at every column
        for (int i = t; i < (all ? CHUNK : listed); i += NT) {
            const int at = all ? i : list[i];
            const uint32_t c = count[at];
            if (c == 0u) continue;
            float y = load1(row_in + v0 + at);
            y = y > 0.0f ? y / rp : y * rp;
            if ((c & ~SEEN) != 0u) y = (y - (float)(c & ~SEEN) * fp) - pp;
            count[at] = ~__float_as_uint(y);
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = t + NT * j, c0 = v0 + i * E;                  // columns c0 .. c0 + E - 1
        if (c0 >= V) break;
        if (vec && c0 >= 0 && c0 + E <= V) {
            uint32_t n[E], any = 0u;
            if (penal) {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const uint4 u = reinterpret_cast<const uint4*>(count)[(i * E + e) >> 2];
                    n[e] = u.x; n[e + 1] = u.y; n[e + 2] = u.z; n[e + 3] = u.w;
                    any |= u.x | u.y | u.z | u.w;
                }
            }
            const uint32_t allow = (uint32_t)(bits[j] >> (c0 & 31)) & ((1u << E) - 1u);
            if (!ahead) {
                if (any == 0u && allow == (1u << E) - 1u) continue;
                x[j].load(row_in + c0);
            }
            float y[E];
            x[j].values(y);
            if (any != 0u) {
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = n[e] != 0u ? __uint_as_float(~n[e]) : y[e];
            }
            if (bias != nullptr) {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const float4_any b = *reinterpret_cast<const float4_any*>(bias + c0 + e);
                    y[e] += b[0]; y[e + 1] += b[1]; y[e + 2] += b[2]; y[e + 3] += b[3];
                }
            }
            if (allow != (1u << E) - 1u) {
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = ((allow >> e) & 1u) != 0u ? y[e] : -INFINITY;
            }
            store16(row_out + c0, y);
        } else {
            for (int e = 0; e < E; ++e) {
                const int v = c0 + e;
                if (v < 0 || v >= V) continue;
                float y = load1(row_in + v);
                if (penal && count[v - v0] != 0u) y = __uint_as_float(~count[v - v0]);
                if (bias != nullptr) y = y + bias[v];
                if (mask != nullptr && ((mask[v >> 5] >> (v & 31)) & 1u) == 0u) y = -INFINITY;
                store1(row_out + v, y);
            }
        }
    }
}

__global__ __launch_bounds__(256) void grammar_next_kernel(const int32_t* __restrict__ next, int64_t n_states, int64_t V,
                                                           const int32_t* __restrict__ state, int64_t R_old, const int32_t* __restrict__ parent,
                                                           const int32_t* __restrict__ tok, int32_t* __restrict__ out, int64_t R) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= R) return;
    const int64_t p = parent != nullptr ? parent[r] : r;
    const int64_t s = p >= 0 && p < R_old ? state[p] : -1, v = tok[r];
    out[r] = s >= 0 && s < n_states && v >= 0 && v < V ? next[s * V + v] : -1;
}

template <typename T>
int adjust_logits(const T* logits, int64_t ld, int64_t R, int64_t V, const tst_logit_rules* a, T* out, int64_t ldo, void* stream,
                  const char* who) {
    TST_REQUIRE(a != nullptr, TST_ERR_ARG, "%s: null rules", who);
    TST_REQUIRE(tst_dims_ok({R, V, a->n_sent, a->n_hist, a->n_prompt, a->n_bias, a->n_masks}), TST_ERR_UNSUPPORTED, "%s: a size exceeds 2^31 - 1", who);
    TST_REQUIRE(R >= 0 && V >= 0 && a->n_sent >= 0 && a->n_hist >= 0 && a->n_prompt >= 0 && a->n_bias >= 0 && a->n_masks >= 0, TST_ERR_ARG,
                "%s: negative size", who);
    constexpr int64_t MOST = 0x7fffffff - 2 * CHUNK_L;      // columns are counted in 32 bits, to the end of the last chunk
    TST_REQUIRE(V <= MOST, TST_ERR_UNSUPPORTED, "%s: columns exceed %lld", who, (long long)MOST);
    TST_REQUIRE(R * V == 0 || (logits && out), TST_ERR_ARG, "%s: null pointer", who);
    TST_REQUIRE(ld >= V && ldo >= V, TST_ERR_ARG, "%s: leading dimensions must hold V columns", who);
    TST_REQUIRE((const void*)logits != (const void*)out || ld == ldo, TST_ERR_ARG, "%s: in place needs one leading dimension", who);
    TST_REQUIRE((a->hist == nullptr && a->prompt == nullptr) || a->params != nullptr, TST_ERR_ARG, "%s: hist and prompt need params", who);
    TST_REQUIRE(a->prompt == nullptr || a->prompt_cu != nullptr, TST_ERR_ARG, "%s: prompt needs prompt_cu", who);
    TST_REQUIRE(a->hist == nullptr || a->ld_hist >= a->n_hist, TST_ERR_ARG, "%s: ld_hist must hold n_hist tokens", who);
    TST_REQUIRE(a->bias == nullptr || a->ld_bias >= V, TST_ERR_ARG, "%s: ld_bias must hold V columns", who);
    TST_REQUIRE(a->mask == nullptr || a->ld_mask >= (V + 31) / 32, TST_ERR_ARG, "%s: ld_mask must hold a bit for each of V columns", who);
    TST_REQUIRE(a->params == nullptr || a->sent != nullptr || a->n_sent >= R, TST_ERR_ARG, "%s: params must hold %lld rows", who, (long long)R);
    if (R == 0 || V == 0) return TST_OK;
    TST_REQUIRE(R <= 0x7fffffff / 4, TST_ERR_UNSUPPORTED, "%s: too many rows", who);
    // Long chunks read a row's tokens less often; few rows are cut finer, to have more workgroups than CUs
    const bool fine = R * ((V + CHUNK_L - 1) / CHUNK_L) < 512;
    const int64_t chunk = fine ? 2048 : CHUNK_L;
    const unsigned chunks = (unsigned)((V + 16 + chunk - 1) / chunk);       // a row may begin up to 7 columns into its first chunk
    for (int64_t r0 = 0; r0 < R; r0 += 65535) {   // grid.y holds at most 65535 rows
        const int64_t n = R - r0 < 65535 ? R - r0 : 65535;
        tst_logit_rules b = *a;
        if (r0 > 0) {   // the rows of this launch start at r0
            if (b.hist) b.hist += r0 * b.ld_hist;
            if (b.hist_len) b.hist_len += r0;
            if (b.bias_row) b.bias_row += r0;
            if (b.mask_row) b.mask_row += r0;
            if (b.sent) b.sent += r0;
            else {
                if (b.params) b.params += 3 * r0;
                if (b.prompt_cu) b.prompt_cu += r0;
                b.n_sent -= r0;
            }
        }
        const dim3 grid(chunks, (unsigned)n);
        if (fine) adjust_logits_kernel<T, 2048, 256><<<grid, 256, 0, (hipStream_t)stream>>>(logits + r0 * ld, ld, (int)V, b, out + r0 * ldo, ldo);
        else adjust_logits_kernel<T, CHUNK_L, NT_L><<<grid, NT_L, 0, (hipStream_t)stream>>>(logits + r0 * ld, ld, (int)V, b, out + r0 * ldo, ldo);
        const int rc = tst_after_launch(who);
        if (rc != TST_OK) return rc;
    }
    return TST_OK;
}

}  // namespace

extern "C" int tst_adjust_logits_f32(const float* logits, int64_t ld, int64_t R, int64_t V, const tst_logit_rules* rules, float* out,
                                     int64_t ldo, void* stream) {
    return adjust_logits<float>(logits, ld, R, V, rules, out, ldo, stream, "tst_adjust_logits_f32");
}
extern "C" int tst_adjust_logits_bf16(const void* logits, int64_t ld, int64_t R, int64_t V, const tst_logit_rules* rules, void* out,
                                      int64_t ldo, void* stream) {
    return adjust_logits<__bf16>((const __bf16*)logits, ld, R, V, rules, (__bf16*)out, ldo, stream, "tst_adjust_logits_bf16");
}

extern "C" int tst_grammar_next(const int32_t* next, int64_t n_states, int64_t V, const int32_t* state, int64_t R_old, const int32_t* parent,
                                const int32_t* tok, int32_t* out, int64_t R, void* stream) {
    TST_REQUIRE(tst_dims_ok({n_states, V, R_old, R}), TST_ERR_UNSUPPORTED, "tst_grammar_next: a size exceeds 2^31 - 1");
    TST_REQUIRE(n_states >= 0 && V >= 0 && R_old >= 0 && R >= 0, TST_ERR_ARG, "tst_grammar_next: negative size");
    TST_REQUIRE(R == 0 || (tok && out && (R_old == 0 || state) && (n_states * V == 0 || next)), TST_ERR_ARG, "tst_grammar_next: null pointer");
    TST_REQUIRE(out == nullptr || out != state, TST_ERR_ARG, "tst_grammar_next: out must not be state");
    if (R == 0) return TST_OK;
    grammar_next_kernel<<<(unsigned)((R + 255) / 256), 256, 0, (hipStream_t)stream>>>(next, n_states, V, state, R_old, parent, tok, out, R);
    return tst_after_launch("tst_grammar_next");
}
