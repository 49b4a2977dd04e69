// Causal attention over whole prompts of different lengths, packed one behind the other, with grouped heads.
#include "tst_common.h"

namespace {

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }

// One wave per (row, head): 64 keys at a time, one per lane for the scores, then each lane sums its elements of the head over them
// with the running maximum and sum of the softmax.
template <typename T>
__global__ __launch_bounds__(64) void attn_prompt_kernel(const T* __restrict__ q, int64_t ldq, const T* __restrict__ k, int64_t ldk,
                                                         const T* __restrict__ v, int64_t ldv, const int32_t* __restrict__ cu, int B,
                                                         T* __restrict__ out, int64_t ldo, int64_t N, int heads, int per_kv, int dh,
                                                         float scale) {
    __shared__ float qs[256], ws[64];
    const int lane = threadIdx.x;
    const int64_t i = blockIdx.x;
    const int h = blockIdx.y, g = h / per_kv;
    // the last sequence that starts at or before i
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= i) lo = mid; else hi = mid;
    }
    const int64_t c0 = cu[lo], c1 = cu[lo + 1];
    if (c0 < 0 || c0 > i || i >= c1) return;
    for (int e = lane; e < dh; e += 64) qs[e] = load1(q + i * ldq + h * dh + e);
    __syncthreads();
    float m = -INFINITY, sum = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t p0 = c0; p0 <= i; p0 += 64) {
        const int64_t p = p0 + lane;
        float score = -INFINITY;
        if (p <= i) {
            float a = 0.0f;
            for (int e = 0; e < dh; ++e) a = __builtin_fmaf(qs[e], load1(k + p * ldk + g * dh + e), a);
            score = a * scale;
        }
        const unsigned long long nan = __ballot(score != score);   // has to reach the result: fmax would drop it
        float top = score;
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        const float mn = nan != 0ull ? __builtin_nanf("") : fmaxf(m, top);
        const float w = p <= i && mn != -INFINITY ? __expf(score - mn) : 0.0f;
        const float keep = m == -INFINITY ? 0.0f : __expf(m - mn);
        float total = w;
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
        sum = sum * keep + total;
        m = mn;
        ws[lane] = w;
        __syncthreads();
        const int n = (int)min((int64_t)64, i - p0 + 1);
        for (int u = 0; u < 4; ++u) {
            const int e = lane + 64 * u;
            if (e < dh) {
                acc[u] *= keep;
                for (int j = 0; j < n; ++j) acc[u] = __builtin_fmaf(ws[j], load1(v + (p0 + j) * ldv + g * dh + e), acc[u]);
            }
        }
        __syncthreads();
    }
    for (int u = 0; u < 4; ++u) {
        const int e = lane + 64 * u;
        if (e < dh) store1(out + i * ldo + h * dh + e, acc[u] / sum);
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
    attn_prompt_kernel<T><<<dim3((unsigned)N, (unsigned)heads), 64, 0, (hipStream_t)stream>>>(q, ldq, k, ldk, v, ldv, cu, (int)B, out, ldo, N,
                                                                                            (int)heads, (int)(heads / kv_heads), (int)dh, scale);
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
