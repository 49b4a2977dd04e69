// Causal attention over whole prompts of different lengths, packed one behind the other, with grouped heads.
//
// A workgroup of four waves takes 128 query rows of one sequence and one head, 32 to a wave, and walks the keys in tiles of KT that all
// four waves read from LDS, with the running maximum and sum of the softmax per query.  On v_mfma_f32_32x32x16_bf16:
//     S^T [KT keys x 32 queries] = K Q^T          O^T [dh x 32 queries] += V^T P^T
// In the accumulator layout a lane holds 16 keys of ONE query, and they are the keys that the second product wants from this lane as
// its B operand (the contraction may visit the keys in any order if both operands agree): the weights never leave their lane, maxima
// and sums cost one exchange between the halves of the wave.  V is read from its row-major tile with the transposing LDS read.
//
// fp32 inputs are split into three bf16 pieces (8 + 8 + 8 bits of significand, exactly the fp32 value) when a tile is staged, and the six
// products of pieces down to 2^-18 of the largest are summed in fp32: what is left out is below 2^-26 of each product, and six bf16
// instructions take 192 cycles where the fp32 matrix instructions would take 512.
#include "tst_common.h"

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) void glb_void;

constexpr int BM = 128;      // query rows per workgroup

union Frag {
    uint32_t u[4];
    uint4 q;
    s16x4 h[2];
    bf16x8 v;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }
__device__ __forceinline__ uint32_t pack2(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2)); }
__device__ __forceinline__ float low_f(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_f(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
__device__ __forceinline__ void store4(__bf16* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(a, b), pack2(c, d));
}

// what a piece that rounds x leaves over; a piece that is infinite or NaN is the whole value
__device__ __forceinline__ float rest(float x, float piece) { return (__float_as_uint(piece) & 0x7f800000u) == 0x7f800000u ? 0.0f : x - piece; }

// eight elements as NP pieces of eight bf16
__device__ __forceinline__ void pieces(const float* p, int have, bool negate, Frag (&f)[3]) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        const float4 v = e < have ? *reinterpret_cast<const float4*>(p + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[e] = v.x; x[e + 1] = v.y; x[e + 2] = v.z; x[e + 3] = v.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = negate ? -x[2 * e] : x[2 * e], b = negate ? -x[2 * e + 1] : x[2 * e + 1];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            f[i].u[e] = pack2(a, b);
            a = rest(a, low_f(f[i].u[e]));
            b = rest(b, high_f(f[i].u[e]));
        }
    }
}
__device__ __forceinline__ void pieces(const __bf16* p, int have, bool negate, Frag (&f)[1]) {
    f[0].q = have >= 8 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
    if (negate) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[0].u[e] ^= 0x80008000u;
    }
}

struct PromptArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t* cu;
    int64_t ldq, ldk, ldv, ldo, N;
    int B, heads, kv_heads, per_kv, dh, tiles;
    float scale2;       // |scale| * log2(e), never 0
    int negate;         // the scale is negative: the query changes its sign
};

// LDS tiles are rows of DH / 8 chunks of 16 bytes.  Chunk c of row r sits at place c ^ swizzle(r), so that the 16 rows that a key fragment
// reads at one c, and the 8 rows x 4 chunks that a value fragment reads, fall on different banks.
template <int DH>
__device__ __forceinline__ int k_swizzle(int r) {
    constexpr int CH = DH / 8, RW = CH >= 16 ? 1 : 16 / CH;
    return (r / RW) & ((CH < 16 ? CH : 16) - 1);
}
template <int DH>
__device__ __forceinline__ int v_swizzle(int r) {
    constexpr int CH = DH / 8;
    return CH >= 16 ? 2 * (r & 7) : (CH == 8 ? 2 * ((r >> 1) & 3) : 0);
}

// One query row by one wave, plainly, reading nothing that the row does not attend to: for rows whose fast result is NaN, because a
// weight of 0 met an infinity or a NaN in a value behind the row, or because the result is one.
template <typename T>
__device__ __forceinline__ void one_row(const PromptArgs& a, int64_t c0, int64_t i, int head, int g) {
    const int lane = threadIdx.x & 63, dh = a.dh;
    const T* q = (const T*)a.q + i * a.ldq + (int64_t)head * dh;
    const T* kb = (const T*)a.k + (int64_t)g * dh;
    const T* vb = (const T*)a.v + (int64_t)g * dh;
    float m = -INFINITY, sum = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t p0 = c0; p0 <= i; p0 += 64) {
        const int64_t p = p0 + lane;
        float s = 0.0f;
        if (p <= i)
            for (int e = 0; e < dh; ++e) s = __builtin_fmaf(load1(q + e), load1(kb + p * a.ldk + e), s);
        s = p <= i ? (a.negate ? -s : s) * a.scale2 : -INFINITY;
        const float top = fmaxf(m, wave_max(s)), base = top == -INFINITY ? 0.0f : top;
        const float w = p <= i ? __builtin_amdgcn_exp2f(s - base) : 0.0f, keep = __builtin_amdgcn_exp2f(m - base);
        sum = sum * keep + wave_sum_butterfly(w);
        m = top;
        const int n = (int)min((int64_t)64, i - p0 + 1);
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] *= keep;
        for (int j = 0; j < n; ++j) {
            const float wj = __shfl(w, j, 64);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (lane + 64 * u < dh) acc[u] = __builtin_fmaf(wj, load1(vb + (p0 + j) * a.ldv + lane + 64 * u), acc[u]);
        }
    }
    T* out = (T*)a.out + i * a.ldo + (int64_t)head * dh;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (lane + 64 * u < dh) store1(out + lane + 64 * u, acc[u] / sum);
}

// DMA: bf16 rows of exactly DH elements go from memory to LDS without registers, two buffers; else through registers, one buffer.
template <typename T, int DH, int KT, bool DMA>
__global__ __launch_bounds__(256) void attn_prompt_kernel(PromptArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 3 : 1;
    constexpr int CH = DH / 8;                       // chunks per row of a tile
    constexpr int PLANE = KT * DH * 2;               // bytes of one piece of a tile
    constexpr int BUF = 2 * NP * PLANE;              // K pieces, then V pieces
    constexpr int KS = DH / 16, MT = DH / 32, NS = KT / 32;
    constexpr int PER = KT * CH / 256;               // chunks of K (and of V) that a thread stages
    __shared__ __attribute__((aligned(16))) unsigned char smem[(DMA ? 2 : 1) * BUF];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int col = lane & 31, h = lane >> 5;

    // Work order: key heads fastest, so that workgroups on one XCD (blockIdx mod 8) share the keys of few heads; then the query heads of
    // a group; then the row tiles, the last (longest) of a sequence first.
    uint32_t id = blockIdx.x;
    const int g = (int)(id % (uint32_t)a.kv_heads);
    id /= (uint32_t)a.kv_heads;
    const int head = g * a.per_kv + (int)(id % (uint32_t)a.per_kv);
    id = (uint32_t)a.tiles - 1u - id / (uint32_t)a.per_kv;
    // Sequence b owns tile numbers from cu[b] / BM + b on: strictly ascending, and always enough of them
    int lo = 0, top_b = a.B;
    while (top_b - lo > 1) {
        const int mid = (lo + top_b) >> 1;
        if ((int64_t)(a.cu[mid] / BM) + mid <= (int64_t)id) lo = mid; else top_b = mid;
    }
    const int64_t c0 = a.cu[lo], c1 = a.cu[lo + 1];
    const int64_t qt = (int64_t)id - (c0 / BM + lo);
    if (c0 < 0 || c1 > a.N || qt < 0 || qt * BM >= c1 - c0) return;      // the whole workgroup
    const int len = (int)(c1 - c0);
    const int q0 = (int)qt * BM, qw = q0 + 32 * w;                       // first row of the workgroup, of this wave (in the sequence)
    const int q_end = min(q0 + BM, len) - 1, w_end = min(qw + 31, len - 1);

    const T* kp = (const T*)a.k + c0 * a.ldk + (int64_t)g * a.dh;
    const T* vp = (const T*)a.v + c0 * a.ldv + (int64_t)g * a.dh;

    // the queries as the B operand: column = query, the half's 8 elements of every step
    Frag q[KS][NP];
    {
        const T* qp = (const T*)a.q + (c0 + min(qw + col, len - 1)) * a.ldq + (int64_t)head * a.dh;
#pragma unroll
        for (int s = 0; s < KS; ++s) pieces(qp + 16 * s + 8 * h, a.dh - (16 * s + 8 * h), a.negate != 0, q[s]);
    }
    f32x16 o[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = -INFINITY, sum = 0.0f;

    // staging: chunk number x = thread + 256 j of a tile is row x / CH, place x % CH
    uint4 stage_k[DMA ? 1 : PER], stage_v[DMA ? 1 : PER];
    float4 stage_k2[NP == 3 ? PER : 1], stage_v2[NP == 3 ? PER : 1];
    auto fetch = [&](int k0, int buf) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int x = threadIdx.x + 256 * j, r = x / CH, c = x % CH;
            const int64_t row = min(k0 + r, len - 1);                    // rows behind the sequence: its last one, weighted 0
            if (DMA) {
                unsigned char* dst = smem + buf * BUF + (w * 64 + 256 * j) * 16;      // + 16 * lane
                __builtin_amdgcn_global_load_lds((glb_void*)(kp + row * a.ldk + 8 * (c ^ k_swizzle<DH>(r))), (lds_void*)dst, 16, 0, 0);
                __builtin_amdgcn_global_load_lds((glb_void*)(vp + row * a.ldv + 8 * (c ^ v_swizzle<DH>(r))), (lds_void*)(dst + PLANE), 16, 0, 0);
            } else {
                const T* sk = kp + row * a.ldk + 8 * c;
                const T* sv = vp + row * a.ldv + 8 * c;
                const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                stage_k[j] = 8 * c < a.dh ? *reinterpret_cast<const uint4*>(sk) : zero;
                stage_v[j] = 8 * c < a.dh ? *reinterpret_cast<const uint4*>(sv) : zero;
                if (NP == 3) {
                    const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                    stage_k2[j] = 8 * c + 4 < a.dh ? *reinterpret_cast<const float4*>(sk + 4) : z;
                    stage_v2[j] = 8 * c + 4 < a.dh ? *reinterpret_cast<const float4*>(sv + 4) : z;
                }
            }
        }
    };
    auto put = [&]() {   // registers -> LDS (not used with DMA)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int x = threadIdx.x + 256 * j, r = x / CH, c = x % CH;
            unsigned char* dk = smem + r * DH * 2 + (c ^ k_swizzle<DH>(r)) * 16;
            unsigned char* dv = smem + NP * PLANE + r * DH * 2 + (c ^ v_swizzle<DH>(r)) * 16;
            if (NP == 1) {
                *reinterpret_cast<uint4*>(dk) = stage_k[j];
                *reinterpret_cast<uint4*>(dv) = stage_v[j];
            } else {
                float x8[8] = {__uint_as_float(stage_k[j].x), __uint_as_float(stage_k[j].y), __uint_as_float(stage_k[j].z),
                               __uint_as_float(stage_k[j].w), stage_k2[j].x, stage_k2[j].y, stage_k2[j].z, stage_k2[j].w};
                float y8[8] = {__uint_as_float(stage_v[j].x), __uint_as_float(stage_v[j].y), __uint_as_float(stage_v[j].z),
                               __uint_as_float(stage_v[j].w), stage_v2[j].x, stage_v2[j].y, stage_v2[j].z, stage_v2[j].w};
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    Frag f, d;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f.u[e] = pack2(x8[2 * e], x8[2 * e + 1]);
                        d.u[e] = pack2(y8[2 * e], y8[2 * e + 1]);
                        x8[2 * e] = rest(x8[2 * e], low_f(f.u[e]));
                        x8[2 * e + 1] = rest(x8[2 * e + 1], high_f(f.u[e]));
                        y8[2 * e] = rest(y8[2 * e], low_f(d.u[e]));
                        y8[2 * e + 1] = rest(y8[2 * e + 1], high_f(d.u[e]));
                    }
                    *reinterpret_cast<uint4*>(dk + i * PLANE) = f.q;
                    *reinterpret_cast<uint4*>(dv + i * PLANE) = d.q;
                }
            }
        }
    };

    // this lane's places in a tile: key row `col`, and value rows 4 h + (lane >> 2) % 4 with 4 elements at 16 ((lane >> 4) & 1) + 4 (lane & 3)
    const int k_row = col * DH * 2, k_sw = k_swizzle<DH>(col);
    const int v_r = 4 * h + ((lane >> 2) & 3);
    const int v_row = v_r * DH * 2 + 8 * (lane & 1), v_sw = v_swizzle<DH>(v_r), v_c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);

    int buf = 0;
    fetch(0, 0);
    for (int k0 = 0; k0 <= q_end; k0 += KT) {
        if (DMA) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // this tile has landed (this wave's share)
            __syncthreads();                                             // everybody's share; and nobody reads the other buffer any more
            if (k0 + KT <= q_end) fetch(k0 + KT, buf ^ 1);
        } else {
            __syncthreads();
            put();
            __syncthreads();
            if (k0 + KT <= q_end) fetch(k0 + KT, 0);
        }
        const unsigned char* kt = smem + buf * BUF;
        const unsigned char* vt = kt + NP * PLANE;
        if (DMA) buf ^= 1;
        if (k0 > w_end || qw >= len) continue;                           // nothing for this wave in the tile
        f32x16 sc[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[n][i] = 0.0f;
            if (n > 0 && k0 + 32 * n > w_end) {                          // keys behind every row of the wave
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[n][i] = -INFINITY;
                continue;
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                Frag k[NP];
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    k[i].q = *reinterpret_cast<const uint4*>(kt + i * PLANE + n * 32 * DH * 2 + k_row + (((2 * s + h) ^ k_sw) << 4));
#pragma unroll
                for (int x = NP - 1; x >= 0; --x)                        // small products first
#pragma unroll
                    for (int i = 0; i <= x; ++i) sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[i].v, q[s][x - i].v, sc[n], 0, 0, 0);
            }
        }
        if (k0 + KT - 1 > qw) {                                          // keys behind some row of the wave
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k0 + 32 * n + 8 * (i >> 2) + 4 * h + (i & 3) > qw + col) sc[n][i] = -INFINITY;
        }
        float top = sc[0][0];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[n][i]);
        top = fmaxf(top, lane_xor<32>(top));
        // The reference point of the weights moves only when the maximum outgrows it by 2^8: the weights stay below 256, far from any
        // limit of fp32, and most tiles skip the rescaling of O.  A first finite score always sets it.
        const bool grow = (top - m) * a.scale2 > 8.0f || (m == -INFINITY && top != -INFINITY);
        if (__ballot(grow) != 0ull) {
            const float next = grow ? top : m;
            const float keep = next == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - next) * a.scale2);
            sum *= keep;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= keep;
            m = next;
        }
        const float base = m == -INFINITY ? 0.0f : m * a.scale2;
        // step s of the second product: 16 keys, the half's 8 in registers 8 (s & 1) .. of the scores of 32-key block s / 2
#pragma unroll
        for (int s = 0; s < KT / 16; ++s) {
            if (s >= 2 && k0 + 16 * s > w_end) break;
            Frag p[NP];
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s >> 1][8 * (s & 1) + i], a.scale2, -base));
                sum += e[i];
            }
#pragma unroll
            for (int x = 0; x < NP; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[x].u[i] = pack2(e[2 * i], e[2 * i + 1]);
                    if (x + 1 < NP) { e[2 * i] -= low_f(p[x].u[i]); e[2 * i + 1] -= high_f(p[x].u[i]); }
                }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                Frag v[NP];
                const int at = s * 16 * DH * 2 + v_row + (((4 * t + v_c) ^ v_sw) << 4);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    v[i].h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + i * PLANE + at));
                    v[i].h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + i * PLANE + at + 8 * DH * 2));
                }
#pragma unroll
                for (int x = NP - 1; x >= 0; --x)
#pragma unroll
                    for (int i = 0; i <= x; ++i) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[i].v, p[x - i].v, o[t], 0, 0, 0);
            }
        }
    }
    if (qw >= len) return;
    sum += lane_xor<32>(sum);
    const bool live = qw + col < len;
    const float inv = 1.0f / sum;
    bool nan = false;
    T* out = (T*)a.out + (c0 + qw + col) * a.ldo + (int64_t)head * a.dh;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int e = 32 * t + 8 * (i >> 2) + 4 * h;
            const float x0 = o[t][i] * inv, x1 = o[t][i + 1] * inv, x2 = o[t][i + 2] * inv, x3 = o[t][i + 3] * inv;
            if (live && e < a.dh) {
                store4(out + e, x0, x1, x2, x3);
                nan |= x0 != x0 || x1 != x1 || x2 != x2 || x3 != x3;
            }
        }
    unsigned long long bad = __ballot(nan);
    for (uint32_t cols = (uint32_t)bad | (uint32_t)(bad >> 32); cols != 0u; cols &= cols - 1u)
        one_row<T>(a, c0, c0 + qw + __builtin_ctz(cols), head, g);
}

template <typename T>
void launch_prompt(const PromptArgs& a, hipStream_t st) {
    const unsigned grid = (unsigned)((int64_t)a.tiles * a.heads);
    if constexpr (sizeof(T) == 2) {
        if (a.dh == 32) attn_prompt_kernel<T, 32, 64, true><<<grid, 256, 0, st>>>(a);
        else if (a.dh == 64) attn_prompt_kernel<T, 64, 64, true><<<grid, 256, 0, st>>>(a);
        else if (a.dh == 128) attn_prompt_kernel<T, 128, 64, true><<<grid, 256, 0, st>>>(a);
        else if (a.dh == 256) attn_prompt_kernel<T, 256, 32, true><<<grid, 256, 0, st>>>(a);
        else if (a.dh < 64) attn_prompt_kernel<T, 64, 64, false><<<grid, 256, 0, st>>>(a);
        else if (a.dh < 128) attn_prompt_kernel<T, 128, 64, false><<<grid, 256, 0, st>>>(a);
        else attn_prompt_kernel<T, 256, 32, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (a.dh <= 64) attn_prompt_kernel<T, 64, 32, false><<<grid, 256, 0, st>>>(a);
        else if (a.dh <= 128) attn_prompt_kernel<T, 128, 32, false><<<grid, 256, 0, st>>>(a);
        else attn_prompt_kernel<T, 256, 32, false><<<grid, 256, 0, st>>>(a);
    }
}

template <typename T>
int attn_prompt(const T* q, int64_t ldq, const T* k, int64_t ldk, const T* v, int64_t ldv, const int32_t* cu, int64_t B, T* out,
                int64_t ldo, int64_t N, int64_t heads, int64_t kv_heads, int64_t dh, float scale, void* stream, const char* who) {
    TST_REQUIRE(tst_dims_ok({B, N, heads, kv_heads, dh}), TST_ERR_UNSUPPORTED, "%s: a size exceeds 2^31 - 1", who);
    TST_REQUIRE(B >= 0 && N >= 0, TST_ERR_ARG, "%s: negative size", who);
    TST_REQUIRE(heads >= 1 && heads <= 4096 && kv_heads >= 1 && heads % kv_heads == 0, TST_ERR_ARG, "%s: heads must be a multiple of kv_heads", who);
    const int64_t unit = 16 / (int64_t)sizeof(T);
    TST_REQUIRE(dh >= unit && dh <= 256 && dh % unit == 0, TST_ERR_UNSUPPORTED, "%s: head size %lld is not a multiple of %d up to 256", who,
                (long long)dh, (int)unit);
    TST_REQUIRE(N == 0 || B == 0 || (q && k && v && cu && out), TST_ERR_ARG, "%s: null pointer", who);
    TST_REQUIRE(ldq % unit == 0 && ldk % unit == 0 && ldv % unit == 0 && ldo % unit == 0 && ldq >= heads * dh && ldo >= heads * dh &&
                    ldk >= kv_heads * dh && ldv >= kv_heads * dh,
                TST_ERR_ARG, "%s: leading dimensions must hold the heads and be multiples of %d", who, (int)unit);
    TST_REQUIRE(tst_aligned16(q) && tst_aligned16(k) && tst_aligned16(v) && tst_aligned16(out), TST_ERR_ARG, "%s: rows must be 16-byte aligned", who);
    if (N == 0 || B == 0) return TST_OK;
    const int64_t tiles = N / BM + B;
    TST_REQUIRE(tiles * heads <= (int64_t)0x7fffffff, TST_ERR_UNSUPPORTED, "%s: too many row tiles", who);
    const PromptArgs a{q, k, v, out, cu, ldq, ldk, ldv, ldo, N, (int)B, (int)heads, (int)kv_heads, (int)(heads / kv_heads), (int)dh, (int)tiles,
                       fmaxf(fabsf(scale) * 1.44269504088896341f, 1e-37f), scale < 0.0f ? 1 : 0};
    launch_prompt<T>(a, (hipStream_t)stream);
    return tst_after_launch(who);
}

}  // namespace

extern "C" int tst_attn_prompt_f32(const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv, const int32_t* cu,
                                   int64_t B, float* out, int64_t ldo, int64_t N, int64_t heads, int64_t kv_heads, int64_t dh, float scale,
                                   void* stream) {
    return attn_prompt<float>(q, ldq, k, ldk, v, ldv, cu, B, out, ldo, N, heads, kv_heads, dh, scale, stream, "tst_attn_prompt_f32");
}
extern "C" int tst_attn_prompt_bf16(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const int32_t* cu,
                                    int64_t B, void* out, int64_t ldo, int64_t N, int64_t heads, int64_t kv_heads, int64_t dh, float scale,
                                    void* stream) {
    return attn_prompt<__bf16>((const __bf16*)q, ldq, (const __bf16*)k, ldk, (const __bf16*)v, ldv, cu, B, (__bf16*)out, ldo, N, heads,
                               kv_heads, dh, scale, stream, "tst_attn_prompt_bf16");
}
