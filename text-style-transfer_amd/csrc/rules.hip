// Rules on the logits of a step: penalties for repeated tokens, biases, grammar masks; and the step of a grammar's states.
#include "tst_common.h"

namespace {

constexpr int CHUNK = 8192;              // columns per workgroup: one 32-bit counter each in LDS
constexpr uint32_t SEEN = 0x80000000u;   // counter bit: the token is in the prompt

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }

// One workgroup per row and chunk of columns: the row's tokens are counted in LDS (integer atomics: the order does not matter),
// then the chunk streams through once.
template <typename T>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const T* logits, int64_t ld, int V, tst_logit_rules a, T* out, int64_t ldo) {
    __shared__ uint32_t count[CHUNK];
    const int t = threadIdx.x;
    const int64_t r = blockIdx.y;
    const int v0 = blockIdx.x * CHUNK, nv = min(CHUNK, V - v0);
    const int64_t s = a.sent != nullptr ? a.sent[r] : r;
    const bool penal = a.params != nullptr && s >= 0 && s < a.n_sent;
    float rp = 1.0f, fp = 0.0f, pp = 0.0f;
    if (penal) {
        rp = a.params[3 * s]; fp = a.params[3 * s + 1]; pp = a.params[3 * s + 2];
        for (int i = t; i < nv; i += 256) count[i] = 0u;
        __syncthreads();
        if (a.prompt != nullptr) {
            const int64_t lo = max((int64_t)a.prompt_cu[s], (int64_t)0), hi = min((int64_t)a.prompt_cu[s + 1], a.n_prompt);
            for (int64_t i = lo + t; i < hi; i += 256) {
                const uint32_t c = (uint32_t)a.prompt[i] - (uint32_t)v0;
                if (c < (uint32_t)nv) atomicOr(&count[c], SEEN);
            }
        }
        if (a.hist != nullptr) {
            const int64_t n = a.hist_len != nullptr ? min((int64_t)a.hist_len[r], a.n_hist) : a.n_hist;
            for (int64_t i = t; i < n; i += 256) {
                const uint32_t c = (uint32_t)a.hist[r * a.ld_hist + i] - (uint32_t)v0;
                if (c < (uint32_t)nv) atomicAdd(&count[c], 1u);
            }
        }
        __syncthreads();
    }
    const int64_t br = a.bias == nullptr ? -1 : (a.bias_row != nullptr ? a.bias_row[r] : 0);
    const int64_t mr = a.mask == nullptr ? -1 : (a.mask_row != nullptr ? a.mask_row[r] : 0);
    const float* bias = br >= 0 && br < a.n_bias ? a.bias + br * a.ld_bias + v0 : nullptr;
    const uint32_t* mask = mr >= 0 && mr < a.n_masks ? a.mask + mr * a.ld_mask + (v0 >> 5) : nullptr;
    for (int i = t; i < nv; i += 256) {
        float y = load1(logits + r * ld + v0 + i);
        if (penal) {
            const uint32_t c = count[i];
            if (c != 0u) y = y > 0.0f ? y / rp : y * rp;
            if ((c & ~SEEN) != 0u) y = (y - (float)(c & ~SEEN) * fp) - pp;
        }
        if (bias != nullptr) y = y + bias[i];
        if (mask != nullptr && ((mask[i >> 5] >> (i & 31)) & 1u) == 0u) y = -INFINITY;
        store1(out + r * ldo + v0 + i, y);
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
    const int chunks = (int)((V + CHUNK - 1) / CHUNK);
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
        adjust_logits_kernel<T><<<dim3((unsigned)chunks, (unsigned)n), 256, 0, (hipStream_t)stream>>>(logits + r0 * ld, ld, (int)V, b, out + r0 * ldo, ldo);
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
