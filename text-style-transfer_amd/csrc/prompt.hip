// Causal attention over whole prompts of different lengths, packed one behind the other, with grouped heads.
//
// A workgroup of four waves (one, for short prompts) takes 128 (32) query rows of one sequence and one head, 32 to a wave, and walks the keys in tiles of KT that all
// four waves read from LDS.  On v_mfma_f32_32x32x16_bf16:
//     S^T [KT keys x 32 queries] = K Q^T          O^T [dh x 32 queries] += V^T P^T
// In the accumulator layout a lane holds 16 keys of ONE query, and they are the keys that the second product wants from this lane as
// its B operand (the contraction may visit the keys in any order if both operands agree): the weights never leave their lane.  V is read
// from its row-major tile with the transposing LDS read.
//
// The softmax needs a reference point per query, not the maximum: exp(s - r) sums and divides the same for every r that neither overflows
// nor underflows it.  r is the largest score of the row's first tile; the score accumulators START at -r, so no subtraction, maximum or
// rescaling of O is left in the loop (one exp2, one product and one sum per weight).  r moves when a sum has outgrown it by 2^60, and
// rows whose result is not finite (64 keys outgrew it by 2^127, a weight of 0 met an infinity) are computed again, plainly.
//
// What bounds it (dh 128, bf16): 64 keys x 32 queries cost a SIMD 1024 cycles of matrix instructions, and the four SIMDs together 1024
// cycles of LDS reads (128 bytes per cycle), so both run full at the limit.  Two prompts of up to 8191 tokens, 16 heads over 4 key heads:
// 479 .. 513 us on different cards, 1.07 .. 1.14 PFLOP/s, the rate of a large library product (29.8 ms plainly).  Measured on the way: a running
// maximum 595 us; 64 queries per wave (half the LDS reads, but one wave per SIMD) 532 us; products of one tile between the exponentials
// of the one before 562 us; workgroups of two waves 583 us; fragments requested where they are used 502 us, 4 keys' and 2 values'
// products ahead 495 us; of 499 us, 29 were the softmax's arithmetic and 126 waiting for LDS.
// 256 prompts of 1 .. 512 tokens, 8 heads of 64: 78 us, 3.4 TB/s, half of it waiting: a workgroup has few tiles, and nearly all of them pass
// the diagonal.  In fp32, 16 prompts of 1 .. 60 tokens, 2 heads of 128: 10.0 us; 8 prompts of 2048, 8
// heads of 64: 142 TFLOP/s, of 128: 129.  (With loads under a condition for heads smaller than the tile 12.6 us, 134 and 107.)
//
// bf16 rounds the weights to bf16 for the second product, off by up to 2^-8 of a weight, and sums the ROUNDED weights (v_dot2, two at a time; fp32
// sums): what is common to a row's weights divides out, so a row that few keys take loses nothing (scores of 30 standard deviations, 8191
// tokens: 1.26e-3 off the exact outputs, 1.99e-3 with the sum of the unrounded weights, 1.21e-3 the result's own rounding).  Rows that all keys
// share remain: 2.0e-3 .. 2.1e-3 in the two cases above, where fp32 weights leave 1.6e-3.  That is a choice for speed: a second piece of the
// weights makes it 1.6e-3, but half as many products again, and those are what bounds this kernel (491 -> 669 us, the ragged prompts 76 -> 84).
//
// fp32 inputs are split into three bf16 pieces (8 + 8 + 8 bits of significand, exactly the fp32 value; the second is at most 2^-8 of the
// first's power of two, the third 2^-17) when a tile is staged, and the six products of pieces i and j with i + j <= 4 are summed in fp32: what
// is left out is at most 2^-24 of each product (the largest found by enumeration 2^-24.04), half a step of fp32, and six bf16
// instructions take 192 cycles where the fp32 matrix instructions would take 512.
#include "tst_common.h"
#include <type_traits>

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;

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

// Eight elements as NP pieces of eight bf16.  What is not finite, or rounds to infinity, leaves a NaN in the second piece, which every product
// passes on: rows that meet it are computed again, plainly.
__device__ __forceinline__ void split8(const float (&x)[8], Frag (&f)[3]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            f[i].u[e] = pack2(a, b);
            a = a - low_f(f[i].u[e]);
            b = b - high_f(f[i].u[e]);
        }
    }
}
// 16 bytes of a head of dh elements at element `at`, zeros behind it, with flipped signs or not.  The load is never under a condition: such
// loads wait for each other.
template <typename T>
__device__ __forceinline__ uint4 query16(const T* head, int at, int dh, uint32_t signs) {
    uint4 v = *reinterpret_cast<const uint4*>(head + min(at, dh - 16 / (int)sizeof(T)));
    const uint32_t keep = at < dh ? 0xffffffffu : 0u;
    v.x = (v.x ^ signs) & keep; v.y = (v.y ^ signs) & keep; v.z = (v.z ^ signs) & keep; v.w = (v.w ^ signs) & keep;
    return v;
}

struct PromptArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t* cu;
    int64_t ldq, ldk, ldv, ldo, N;
    int B, heads, kv_heads, per_kv, dh, tiles;
    float scale2;       // |scale| * log2(e), never 0
    int negate;         // the scale is negative: the query changes its sign
    int by_rows;        // work order
};

// 16 bytes per lane from base + offset to LDS address lds + 16 * lane.  As assembly, because the compiler would make every later LDS read
// wait for it, not knowing that those read the other buffer; it writes no register, and the kernel waits for it before the barrier that
// opens its buffer.
__device__ __forceinline__ void dma16(uint32_t lds, const void* base, uint32_t offset) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(lds), "v"(offset), "s"(base) : "memory");
}

// LDS tiles are rows of DH / 8 chunks of 16 bytes.  Chunk c of row r sits at place c ^ swizzle(r), so that what an LDS read fetches in one
// clock falls on different banks, whether that is 128 bytes of 32 banks or 256 of 64: 8 or 16 rows at one chunk for a key fragment, 4
// rows at 2 or 4 chunks for a value fragment.  (Rows of 256 bytes or more: all rows start at bank 0; of 128: every second; of 64: fourth.)
template <int DH>
__device__ __forceinline__ int k_swizzle(int r) {
    constexpr int CH = DH / 8;
    return CH >= 16 ? r & 15 : (CH == 8 ? (r & 6) | ((r ^ (r >> 3)) & 1) : (((r >> 1) ^ (r >> 3)) & 1) | ((r >> 1) & 2));
}
template <int DH>
__device__ __forceinline__ int v_swizzle(int r) {
    constexpr int CH = DH / 8;
    return CH >= 16 ? 2 * (r & 3) + 8 * (r & 1) : (CH == 8 ? 2 * (r & 3) : r & 2);
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
// PACKED: the waves of a workgroup take the same 32 rows of adjacent heads that share a key head.
template <typename T, int DH, int KT, bool DMA, int WAVES, bool PACKED>
__global__ __launch_bounds__(64 * WAVES, DMA && DH <= 128 ? 2 : 1) void attn_prompt_kernel(PromptArgs a) {
    constexpr int NT = 64 * WAVES, BM = PACKED ? 32 : 32 * WAVES;      // threads, rows per workgroup
    constexpr int NP = sizeof(T) == 4 ? 3 : 1;
    constexpr int CH = DH / 8;                       // chunks per row of a tile
    constexpr int PLANE = KT * DH * 2;               // bytes of one piece of a tile
    constexpr int BUF = 2 * NP * PLANE;              // K pieces, then V pieces
    constexpr int KS = DH / 16, MT = DH / 32, NS = KT / 32;
    constexpr int PER = KT * CH / NT;                // chunks of K (and of V) that a thread stages
    constexpr bool AHEAD = (DMA || NP == 3) && DH <= 128;         // fragments are requested KD (VD) products before they are wanted
    constexpr int KD = AHEAD ? (NP == 3 ? 2 : 4) : 1, VD = AHEAD ? 2 : 1;
    constexpr bool DOUBLE = DMA && WAVES > 1;        // two tiles in LDS: the next one lands while this one is worked on
    __shared__ __attribute__((aligned(16))) unsigned char smem[(DOUBLE ? 2 : 1) * BUF];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int col = lane & 31, h = lane >> 5;

    // Work order (workgroup i runs on XCD i mod 8).  Long sequences: key heads fastest, so that an XCD's L2 holds the keys of few heads; then
    // the query heads of a group; then the row tiles.  Short ones, whose keys fit there together: all heads of a row tile on one XCD, which
    // so reads whole rows.  (Prompts of 1 .. 512 tokens, 8 heads of 64: 78 us by rows, 82.5 by heads; of 8191, 16 heads of 128: 513 and 484.)
    // The last, longest row tiles of a sequence come first.
    uint32_t id = blockIdx.x;
    int head;                                        // PACKED: the first of WAVES adjacent ones
    const uint32_t heads = (uint32_t)a.heads / (PACKED ? WAVES : 1), per_kv = (uint32_t)a.per_kv / (PACKED ? WAVES : 1);
    if (a.by_rows) {
        const uint32_t xcd = id & 7u;
        id >>= 3;
        head = (int)(id % heads);
        id /= heads;
        id = id * 8u + ((xcd + 3u * id) & 7u);   // rotated, so that tiles without rows, every second or third for some lengths, meet every XCD
        if (id >= (uint32_t)a.tiles) return;
    } else {
        const int key_head = (int)(id % (uint32_t)a.kv_heads);
        id /= (uint32_t)a.kv_heads;
        head = key_head * (int)per_kv + (int)(id % per_kv);
        id /= per_kv;
    }
    if (PACKED) head *= WAVES;
    const int g = head / a.per_kv;
    if (PACKED) head += w;
    id = (uint32_t)a.tiles - 1u - id;
    // Sequence b owns tile numbers from cu[b] / BM + b on: strictly ascending, and always enough of them.  A search by 64 probes at once, the
    // last of which also hold the sequence's ends: one load for up to 64 sequences, two for 4096.
    int lo = 0, begin, end;
    for (int n = a.B;;) {
        const int step = (n + 63) >> 6, at = lo + lane * step;
        const int probe = lane * step <= n ? a.cu[at] : 0;
        const bool starts = lane * step < n && (int64_t)(probe / BM) + at <= (int64_t)id;
        const int count = max(__builtin_popcountll(__ballot(starts)), 1) - 1;
        lo += count * step;
        if (step == 1) {
            begin = __builtin_amdgcn_readlane(probe, count);
            end = count < 63 ? __builtin_amdgcn_readlane(probe, count + 1) : a.cu[lo + 1];
            break;
        }
        n = min(step, n - count * step);
    }
    const int64_t c0 = begin, c1 = end;
    const int64_t qt = (int64_t)id - (c0 / BM + lo);
    if (c0 < 0 || c1 > a.N || qt < 0 || qt * BM >= c1 - c0) return;      // the whole workgroup
    const int len = (int)(c1 - c0);
    const int q0 = (int)qt * BM, qw = q0 + (PACKED ? 0 : 32 * w), row = qw + col;      // workgroup's, wave's first, lane's row
    const int q_end = min(q0 + BM, len) - 1, w_end = min(qw + 32, len) - 1;

    const T* kp = (const T*)a.k + c0 * a.ldk + (int64_t)g * a.dh;
    const T* vp = (const T*)a.v + c0 * a.ldv + (int64_t)g * a.dh;

    // the queries as the B operand: column = query, the half's 8 elements of every step; fp32 heads of more than 128 elements keep them whole
    // (256 registers of pieces would not leave room for O) and split them at every use
    constexpr bool WHOLE = NP == 3 && DH > 128;
    Frag q[KS][WHOLE ? 2 : NP];
    {
        const T* qp = (const T*)a.q + (c0 + min(row, len - 1)) * a.ldq + (int64_t)head * a.dh;
        const uint32_t signs = a.negate == 0 ? 0u : (NP == 3 ? 0x80000000u : 0x80008000u);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int at = 16 * s + 8 * h;
            if constexpr (NP == 1) {
                q[s][0].q = query16(qp, at, a.dh, signs);
            } else if constexpr (WHOLE) {
                q[s][0].q = query16(qp, at, a.dh, signs);
                q[s][1].q = query16(qp, at + 4, a.dh, signs);
            } else {
                const uint4 u = query16(qp, at, a.dh, signs), v = query16(qp, at + 4, a.dh, signs);
                const float e8[8] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w),
                                     __uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
                split8(e8, q[s]);
            }
        }
    }
    f32x16 o[MT], start;                             // start: where score accumulators start from, minus the query's reference point
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) start[i] = 0.0f;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;

    // staging: chunk number x = thread + NT j of a tile is row x / CH, place x % CH
    u32x4 stage_k[DMA ? 1 : PER], stage_v[DMA ? 1 : PER];
    float4 stage_k2[NP == 3 ? PER : 1], stage_v2[NP == 3 ? PER : 1];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)smem;
    const int wu = __builtin_amdgcn_readfirstlane(w);
    // A lane's byte offsets within a whole tile never change: the tile's own address is scalar.  Chunks behind the head read its last elements
    // again: the query is 0 there, and such outputs are not stored.
    uint32_t off_k[PER], off_v[PER];
    constexpr int PIECE = 16 / (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int x = threadIdx.x + NT * j, r = x / CH, c = x % CH;
        off_k[j] = (uint32_t)(r * (int)a.ldk + (DMA ? 8 * (c ^ k_swizzle<DH>(r)) : min(8 * c, a.dh - PIECE))) * (uint32_t)sizeof(T);
        off_v[j] = (uint32_t)(r * (int)a.ldv + (DMA ? 8 * (c ^ v_swizzle<DH>(r)) : min(8 * c, a.dh - PIECE))) * (uint32_t)sizeof(T);
    }
    auto fetch = [&](int k0, int buf) {
        const unsigned char* tk = reinterpret_cast<const unsigned char*>(kp + (int64_t)k0 * a.ldk);
        const unsigned char* tv = reinterpret_cast<const unsigned char*>(vp + (int64_t)k0 * a.ldv);
        const bool whole = k0 + KT <= len;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int x = threadIdx.x + NT * j, r = x / CH, c = x % CH;
            uint32_t ok = off_k[j], ov = off_v[j];
            if (!whole) {                                                // rows behind the sequence: its last one, weighted 0
                const int back = max(k0 + r - (len - 1), 0);
                ok -= (uint32_t)(back * (int)a.ldk) * (uint32_t)sizeof(T);
                ov -= (uint32_t)(back * (int)a.ldv) * (uint32_t)sizeof(T);
            }
            if (DMA) {
                const uint32_t dst = lds0 + buf * BUF + (wu * 64 + NT * j) * 16;
                dma16(dst, tk, ok);
                dma16(dst + PLANE, tv, ov);
            } else {
                const unsigned char* sk = tk + (int64_t)(int32_t)ok;
                const unsigned char* sv = tv + (int64_t)(int32_t)ov;
                stage_k[j] = *reinterpret_cast<const u32x4*>(sk);
                stage_v[j] = *reinterpret_cast<const u32x4*>(sv);
                if (NP == 3) {
                    const int second = 8 * c + 4 < a.dh ? 16 : 0;
                    stage_k2[j] = *reinterpret_cast<const float4*>(sk + second);
                    stage_v2[j] = *reinterpret_cast<const float4*>(sv + second);
                }
            }
        }
    };
    auto put = [&]() {   // registers -> LDS (not used with DMA)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int x = threadIdx.x + NT * j, r = x / CH, c = x % CH;
            unsigned char* dk = smem + r * DH * 2 + (c ^ k_swizzle<DH>(r)) * 16;
            unsigned char* dv = smem + NP * PLANE + r * DH * 2 + (c ^ v_swizzle<DH>(r)) * 16;
            if (NP == 1) {
                *reinterpret_cast<u32x4*>(dk) = stage_k[j];
                *reinterpret_cast<u32x4*>(dv) = stage_v[j];
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
                        x8[2 * e] = x8[2 * e] - low_f(f.u[e]);
                        x8[2 * e + 1] = x8[2 * e + 1] - high_f(f.u[e]);
                        y8[2 * e] = y8[2 * e] - low_f(d.u[e]);
                        y8[2 * e + 1] = y8[2 * e + 1] - high_f(d.u[e]);
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
            if (DOUBLE && k0 + KT <= q_end) fetch(k0 + KT, buf ^ 1);
        } else {
            __syncthreads();
            put();
            __syncthreads();
            if (k0 + KT <= q_end) fetch(k0 + KT, 0);
        }
        const unsigned char* kt = smem + buf * BUF;
        const unsigned char* vt = kt + NP * PLANE;
        if (DOUBLE) buf ^= 1;
        if (k0 > w_end || qw >= len) continue;                           // nothing for this wave in the tile
        // EDGE: the wave's first tile (which sets the reference point) and tiles that end behind some row of it
        auto tile = [&](auto edge) {
            constexpr bool EDGE = decltype(edge)::value;
            const auto beyond = [&](int key) { return EDGE && k0 + key > w_end; };      // keys behind every row of the wave
            f32x16 sc[NS];                                               // scores, then weights
            Frag k[KD][NP], v[VD][NP];
            const auto read_key = [&](Frag (&f)[NP], int n, int s) {
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    f[i].q = *reinterpret_cast<const uint4*>(kt + i * PLANE + n * 32 * DH * 2 + k_row + (((2 * s + h) ^ k_sw) << 4));
            };
            const auto read_value = [&](Frag (&f)[NP], int s, int t) {
                const int at = s * 16 * DH * 2 + v_row + (((4 * t + v_c) ^ v_sw) << 4);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    f[i].h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + i * PLANE + at));
                    f[i].h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + i * PLANE + at + 8 * DH * 2));
                }
            };
            // Fragments are requested KD (VD) products ahead: an LDS read takes several products' time, and left alone the compiler asks for
            // one or two at a time.
#pragma unroll
            for (int x = 0; x < KD; ++x) read_key(k[x], x / KS, x % KS);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                if (n > 0 && beyond(32 * n)) continue;   // its requested fragments go unused
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int at = n * KS + s;
                    Frag (&f)[NP] = k[at % KD];
                    Frag split[WHOLE ? NP : 1];
                    if constexpr (WHOLE) {
                        float e8[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            uint32_t u = q[s][e >> 2].u[e & 3];
                            asm volatile("" : "+v"(u));              // or the compiler would split them all before the loop
                            e8[e] = __uint_as_float(u);
                        }
                        split8(e8, split);
                    }
                    const auto& qs = [&]() -> const auto& { if constexpr (WHOLE) return split; else return q[s]; }();
#pragma unroll
                    for (int x = NP - 1; x >= 0; --x)                // small products first
#pragma unroll
                        for (int i = 0; i <= x; ++i)
                            sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i].v, qs[x - i].v,
                                                                               s == 0 && x == NP - 1 && i == 0 ? start : sc[n], 0, 0, 0);
                    if (at + KD < NS * KS) read_key(f, (at + KD) / KS, (at + KD) % KS);
                    if (AHEAD) __builtin_amdgcn_sched_barrier(0);
                }
                if (EDGE && k0 + 32 * n + 31 > qw) {
                    const int own = row - k0 - 32 * n - 4 * h;           // the row's own key, counted from this lane's first
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (8 * (i >> 2) + (i & 3) > own) sc[n][i] = -INFINITY;
                }
                // Scores are relative to the reference point, which the accumulators start from: the largest of the first 32 keys'.
                if (EDGE && n == 0 && k0 == 0) {
                    float top = sc[0][0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[0][i]);
                    top = fmaxf(top, lane_xor<32>(top));
                    top = top == -INFINITY ? 0.0f : top;                 // no finite score yet: any point will do
#pragma unroll
                    for (int i = 0; i < 16; ++i) sc[0][i] -= top;
#pragma unroll
                    for (int i = 0; i < 16; ++i) start[i] = -top;
                }
            }
            const int steps = beyond(32) ? 2 : KT / 16;
#pragma unroll
            for (int x = 0; x < VD; ++x) read_value(v[x], x / MT, x % MT);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
            Frag p[KT / 16][NP];
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                if (n > 0 && beyond(32 * n)) continue;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[n][i] = __builtin_amdgcn_exp2f(sc[n][i] * a.scale2);
                    if (NP == 3) sum += sc[n][i];
                }
                // step s of the second product: 16 keys, the half's 8 in registers 8 (s & 1) .. of the weights of 32-key block s / 2
#pragma unroll
                for (int s = 2 * n; s < 2 * n + 2; ++s)
#pragma unroll
                    for (int x = 0; x < NP; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = 8 * (s & 1) + 2 * i;
                            p[s][x].u[i] = pack2(sc[n][at], sc[n][at + 1]);
                            if (NP == 1)                              // the sum of the weights as they are multiplied
                                sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p[s][x].u[i]), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
                            if (x + 1 < NP) {
                                sc[n][at] -= low_f(p[s][x].u[i]);
                                sc[n][at + 1] -= high_f(p[s][x].u[i]);
                            }
                        }
            }
#pragma unroll
            for (int s = 0; s < KT / 16; ++s) {
                if (s >= 2 && s >= steps) break;
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const int at = s * MT + t;
                    Frag (&f)[NP] = v[at % VD];
#pragma unroll
                    for (int x = NP - 1; x >= 0; --x)
#pragma unroll
                        for (int i = 0; i <= x; ++i) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i].v, p[s][x - i].v, o[t], 0, 0, 0);
                    if (at + VD < KT / 16 * MT) read_value(f, (at + VD) / MT, (at + VD) % MT);
                }
            }
        };
        if (k0 == 0 || k0 + KT - 1 > qw) tile(std::true_type{});
        else tile(std::false_type{});
        if (DMA && !DOUBLE && k0 + KT <= q_end) {                        // one buffer: the wave's reads of this tile are back before it is written
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            fetch(k0 + KT, 0);
        }
        // The reference point moves when a sum has outgrown it by 2^60: far from any limit of fp32, and rare.  (64 keys that outgrow it by 2^127
        // overflow; their rows are computed again at the end.)  It moves after every 64 keys and after the wave's last ones, whatever a tile
        // holds: the same bits from every form of this kernel.
        if ((KT % 64 == 0 || ((k0 + KT) & 63) == 0 || k0 + KT > w_end) && __ballot(sum > 0x1p60f) != 0ull) {
            const int by = __builtin_amdgcn_frexp_expf(fmaxf(fmaxf(sum, lane_xor<32>(sum)), 1.0f));     // (a factor 2^-by could be subnormal)
            const float raw = (float)by / a.scale2;
            sum = __builtin_amdgcn_ldexpf(sum, -by);
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] = __builtin_amdgcn_ldexpf(o[t][i], -by);
#pragma unroll
            for (int i = 0; i < 16; ++i) start[i] -= raw;
        }
    }
    if (qw >= len) return;
    const float total = sum + lane_xor<32>(sum);
    const float inv = 1.0f / total;
    bool odd = !(total < INFINITY);
    uint32_t word[2][2];
    T* out = (T*)a.out + (c0 + row) * a.ldo + (int64_t)head * a.dh;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = o[t][i + u] * inv;
            const float none = (x[0] - x[0]) + (x[1] - x[1]) + (x[2] - x[2]) + (x[3] - x[3]);      // 0, or NaN if one is not finite
            odd |= none != 0.0f;
            const int e = 32 * t + 8 * (i >> 2) + 4 * h;
            if constexpr (NP == 3) {
                if (row < len && e < a.dh) *reinterpret_cast<float4*>(out + e) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
                // the halves of the wave hold four elements each of a chunk of 16 bytes: of two chunks each takes one whole
                word[i / 4 & 1][0] = pack2(x[0], x[1]);
                word[i / 4 & 1][1] = pack2(x[2], x[3]);
                if (i / 4 & 1) {
                    const auto p0 = __builtin_amdgcn_permlane32_swap(word[0][0], word[1][0], false, false);
                    const auto p1 = __builtin_amdgcn_permlane32_swap(word[0][1], word[1][1], false, false);
                    const int chunk = 32 * t + 2 * i - 8 + 8 * h;
                    if (row < len && chunk < a.dh) *reinterpret_cast<uint4*>(out + chunk) = make_uint4(p0[0], p1[0], p0[1], p1[1]);
                }
            }
        }
    unsigned long long bad = __ballot(odd && row < len);
    for (uint32_t cols = (uint32_t)bad | (uint32_t)(bad >> 32); cols != 0u; cols &= cols - 1u)
        one_row<T>(a, c0, c0 + qw + __builtin_ctz(cols), head, g);
}

template <typename T, int DH, int KT, bool DMA, int WAVES = 4, bool PACKED = false>
int launch_one(PromptArgs a, hipStream_t st, const char* who) {
    constexpr int BM = PACKED ? 32 : 32 * WAVES;
    const int64_t tiles = a.N / BM + a.B;                                   // sequence b owns tiles cu[b] / BM + b ..
    a.by_rows = a.N / a.B * a.kv_heads * a.dh * 2 * (int64_t)sizeof(T) <= (1 << 21);
    const int64_t groups = (a.by_rows ? (tiles + 7) / 8 * 8 : tiles) * (a.heads / (PACKED ? WAVES : 1));
    TST_REQUIRE(groups <= (int64_t)0x7fffffff, TST_ERR_UNSUPPORTED, "%s: too many row tiles", who);
    a.tiles = (int)tiles;
    attn_prompt_kernel<T, DH, KT, DMA, WAVES, PACKED><<<(unsigned)groups, 64 * WAVES, 0, st>>>(a);
    return tst_after_launch(who);
}

template <typename T>
int launch_prompt(const PromptArgs& a, hipStream_t st, const char* who) {
    // More workgroups of four waves of rows than the GPU holds at once (those of 128 elements and more in fp32, of 256 in bf16: one per CU)
    const bool many = (a.N / 128 + a.B) * a.heads > (a.dh > (sizeof(T) == 4 ? 64 : 128) ? 256 : 512);
    // Such calls with few rows per prompt, where most waves would have none: the waves take four heads that share a key head instead, which
    // also stages the keys (in fp32: splits them) once for the four.  Prompts of 16 tokens, four waves of rows / packed: fp32, 16 heads over 4 of
    // 128, 16 prompts 13.1 / 8.3 us, 256 prompts 102 / 35; 8 over 2 of 64, 72 prompts 9.1 / 6.0; bf16, 4 over 1 of 256, 72 prompts 11.5 / 7.9.  Of 96
    // tokens: 26.5 / 17.1, 214 / 158, 19.4 / 17.8, 20.1 / 24.9.  Calls that fit at once lose (fp32, 8 over 2 of 64, 16 of 16: 5.0 / 5.4).
    const bool packed = many && a.per_kv % 4 == 0 && a.N / a.B <= (sizeof(T) == 4 ? 96 : 64);
    if constexpr (sizeof(T) == 2) {
        // Prompts of a few rows: one wave per workgroup, one tile of 32 keys in LDS, so that many are at work (256 prompts, 32 heads over 8 of
        // 128: 2 tokens each 19 us, 62 with four waves; 32 tokens 32 and 74; 64 tokens 86 and 110; 96 tokens 135 and 150, but of 8 heads of 64
        // 27 and 22).  A row's sums run over the same keys in the same order, and its reference point moves at the same keys, either way.
        if (a.N / a.B <= 64) {
            if (a.dh == 32) return launch_one<T, 32, 32, true, 1>(a, st, who);
            if (a.dh == 64) return launch_one<T, 64, 32, true, 1>(a, st, who);
            if (a.dh == 128) return launch_one<T, 128, 32, true, 1>(a, st, who);
        }
        if (packed && a.dh == 256) return launch_one<T, 256, 32, true, 4, true>(a, st, who);
        if (a.dh == 32) return launch_one<T, 32, 64, true>(a, st, who);
        if (a.dh == 64) return launch_one<T, 64, 64, true>(a, st, who);
        if (a.dh == 128) return launch_one<T, 128, 64, true>(a, st, who);
        if (a.dh == 256) return launch_one<T, 256, 32, true>(a, st, who);
        if (a.dh < 64) return launch_one<T, 64, 64, false>(a, st, who);
        if (a.dh < 128) return launch_one<T, 128, 64, false>(a, st, who);
        return launch_one<T, 256, 32, false>(a, st, who);
    } else {
        if (packed && a.dh > 32) {                       // (not for heads of 256 elements: registers)
            if (a.dh <= 64) return launch_one<T, 64, 32, false, 4, true>(a, st, who);
            if (a.dh <= 128) return launch_one<T, 128, 32, false, 4, true>(a, st, who);
        }
        // One wave per workgroup as in bf16, but here a tile costs its wave the splitting into pieces too: only where there are more workgroups
        // than the GPU holds at once (256 prompts of 32 tokens, 16 heads of 128: 60 us, 105 with four waves, of 64 tokens 142 and 162, of 96 238 and
        // 229; 8 heads of 64: 18 and 25, 32 and 36, 51 and 48; 16 prompts of 32 tokens, 8 heads of 64: 5.6 and 5.1).
        if (many && a.N / a.B <= 64) {
            if (a.dh <= 32) return launch_one<T, 32, 32, false, 1>(a, st, who);
            if (a.dh <= 64) return launch_one<T, 64, 32, false, 1>(a, st, who);
            if (a.dh <= 128) return launch_one<T, 128, 32, false, 1>(a, st, who);
        }
        if (a.dh <= 32) return launch_one<T, 32, 64, false>(a, st, who);
        // 64 keys per tile where they leave two workgroups to a CU (8 prompts of 2048, 8 heads of 64: 241 us, with 32 keys 273; heads of 128: no gain)
        if (a.dh <= 64) return launch_one<T, 64, 64, false>(a, st, who);
        if (a.dh <= 128) return launch_one<T, 128, 32, false>(a, st, who);
        return launch_one<T, 256, 32, false>(a, st, who);
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
    TST_REQUIRE(scale - scale == 0.0f, TST_ERR_ARG, "%s: scale is not finite", who);
    TST_REQUIRE(N == 0 || B == 0 || (q && k && v && cu && out), TST_ERR_ARG, "%s: null pointer", who);
    TST_REQUIRE(ldq % unit == 0 && ldk % unit == 0 && ldv % unit == 0 && ldo % unit == 0 && ldq >= heads * dh && ldo >= heads * dh &&
                    ldk >= kv_heads * dh && ldv >= kv_heads * dh,
                TST_ERR_ARG, "%s: leading dimensions must hold the heads and be multiples of %d", who, (int)unit);
    TST_REQUIRE(tst_aligned16(q) && tst_aligned16(k) && tst_aligned16(v) && tst_aligned16(out), TST_ERR_ARG, "%s: rows must be 16-byte aligned", who);
    if (N == 0 || B == 0) return TST_OK;
    TST_REQUIRE(ldk <= (1 << 22) && ldv <= (1 << 22), TST_ERR_UNSUPPORTED, "%s: a leading dimension of k or v exceeds 2^22", who);   // offsets in a tile are 32-bit
    const PromptArgs a{q, k, v, out, cu, ldq, ldk, ldv, ldo, N, (int)B, (int)heads, (int)kv_heads, (int)(heads / kv_heads), (int)dh, 0,
                       fmaxf(fabsf(scale) * 1.44269504088896341f, 1e-37f), scale < 0.0f ? 1 : 0, 0};
    return launch_prompt<T>(a, (hipStream_t)stream, who);
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
