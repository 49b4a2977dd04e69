// A key / value cache in 4 bits: stored, read back, and attended to by one query row per sequence.
//
// Format (declared with tst_cache4): 32 elements of a head share a power of two; an element is a 4-bit float (sign, two exponent
// bits, one mantissa bit).  Scaling by a power of two is exact, so which code an element gets is decided without any rounding
// before the one that the format itself makes, in fp32 as in 64 bits.
#include "tst_common.h"

namespace {

struct Cache {
    uint8_t *kc, *ks, *vc, *vs;
    int64_t slots;      // pages * page
    int page_shift, kv_heads, dh;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }

// the scale byte of a group from the bits of its largest magnitude: with max = f * 2^(B - 127), 1 <= f < 2, the smallest E with
// max <= 6 * 2^E = 1.5 * 2^(E + 2) is B - 129, one more if f > 1.5; bytes 1 .. 253 (E -126 .. 126), 255 for NaN and infinities
__device__ __forceinline__ int scale_byte(uint32_t top_bits) {
    if (top_bits >= 0x7f800000u) return 255;
    const int s = (int)(top_bits >> 23) - 2 + ((top_bits & 0x7fffffu) > 0x400000u ? 1 : 0);
    return s < 1 ? 1 : s;
}
// 2^-(s - 127) as a float, s in 1 .. 253
__device__ __forceinline__ float inverse_scale(int s) { return __uint_as_float((uint32_t)(254 - s) << 23); }

// the code of y = x * 2^-E, |y| <= 6: nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code
__device__ __forceinline__ uint32_t code_of(float y) {
    const float a = fabsf(y);
    const uint32_t m = (uint32_t)(a > 0.25f) + (uint32_t)(a >= 0.75f) + (uint32_t)(a > 1.25f) + (uint32_t)(a >= 1.75f) +
                       (uint32_t)(a > 2.5f) + (uint32_t)(a >= 3.5f) + (uint32_t)(a > 5.0f);
    return m | (y < 0.0f ? 8u : 0u);
}
// the value of a code
__device__ __forceinline__ float value_of(uint32_t c) {
    const uint32_t e = (c >> 1) & 3u, m = c & 1u;
    const float v = e == 0u ? (m != 0u ? 0.5f : 0.0f) : __uint_as_float(((e + 126u) << 23) | (m << 22));
    return (c & 8u) != 0u ? -v : v;
}
__device__ __forceinline__ float scale_of(uint32_t s) { return s == 255u ? __builtin_nanf("") : __uint_as_float((s < 1u ? 1u : s) << 23); }

// One lane per (token, group of 32 elements): lanes of a wave are consecutive tokens, so that the bytes of the token-minor value
// codes are written side by side; the 4 waves of a workgroup take 4 adjacent groups of the same 64 tokens.
template <typename T>
__global__ __launch_bounds__(256) void cache4_write_kernel(Cache c, const T* __restrict__ k, int64_t ldk, const T* __restrict__ v,
                                                           int64_t ldv, const int32_t* __restrict__ slots, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int groups = c.dh >> 5;
    const int hg = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (i >= n || hg >= c.kv_heads * groups) return;
    const int64_t slot = slots[i];
    if (slot < 0 || slot >= c.slots) return;
    const int h = hg / groups, g = hg - h * groups;
    const int page = 1 << c.page_shift;
    const int64_t ph = (slot >> c.page_shift) * c.kv_heads + h;
    const int tok = (int)(slot & (page - 1));
    const T* src = (blockIdx.z == 0 ? k + i * ldk : v + i * ldv) + h * c.dh + g * 32;
    float x[32];
    uint32_t top = 0;
    for (int e = 0; e < 32; ++e) {
        x[e] = load1(src + e);
        const uint32_t a = __float_as_uint(x[e]) & 0x7fffffffu;
        top = top > a ? top : a;
    }
    const int s = scale_byte(top);
    const float inv = inverse_scale(s == 255 ? 127 : s);
    uint8_t* codes = blockIdx.z == 0 ? c.kc + (ph * page + tok) * (c.dh >> 1) + g * 16 : c.vc + (ph * (c.dh >> 1) + g * 16) * page + tok;
    const int64_t step = blockIdx.z == 0 ? 1 : page;
    for (int e = 0; e < 16; ++e) codes[e * step] = (uint8_t)(code_of(x[2 * e] * inv) | (code_of(x[2 * e + 1] * inv) << 4));
    uint8_t* sc = blockIdx.z == 0 ? c.ks + (ph * page + tok) * groups + g : c.vs + (ph * groups + g) * page + tok;
    *sc = (uint8_t)s;
}

template <typename T>
__global__ __launch_bounds__(256) void cache4_read_kernel(Cache c, const int32_t* __restrict__ slots, T* __restrict__ k, int64_t ldk,
                                                          T* __restrict__ v, int64_t ldv, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int groups = c.dh >> 5;
    const int hg = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (i >= n || hg >= c.kv_heads * groups) return;
    const int64_t slot = slots[i];
    const int h = hg / groups, g = hg - h * groups;
    T* dst = (blockIdx.z == 0 ? k + i * ldk : v + i * ldv) + h * c.dh + g * 32;
    if (slot < 0 || slot >= c.slots) {
        for (int e = 0; e < 32; ++e) store1(dst + e, 0.0f);
        return;
    }
    const int page = 1 << c.page_shift;
    const int64_t ph = (slot >> c.page_shift) * c.kv_heads + h;
    const int tok = (int)(slot & (page - 1));
    const uint8_t* codes = blockIdx.z == 0 ? c.kc + (ph * page + tok) * (c.dh >> 1) + g * 16 : c.vc + (ph * (c.dh >> 1) + g * 16) * page + tok;
    const int64_t step = blockIdx.z == 0 ? 1 : page;
    const float f = scale_of(blockIdx.z == 0 ? c.ks[(ph * page + tok) * groups + g] : c.vs[(ph * groups + g) * page + tok]);
    for (int e = 0; e < 16; ++e) {
        const uint32_t b = codes[e * step];
        store1(dst + 2 * e, value_of(b & 15u) * f);
        store1(dst + 2 * e + 1, value_of(b >> 4) * f);
    }
}

// One wave per (row, head): 64 tokens at a time, one per lane for the scores, then each lane sums its elements of the head over
// them with the running maximum and sum of the softmax.
template <typename T>
__global__ __launch_bounds__(64) void attn_cache4_kernel(Cache c, const T* __restrict__ q, int64_t ldq, const int32_t* __restrict__ table,
                                                         int64_t width, int64_t n_seq, const int32_t* __restrict__ seq,
                                                         const int32_t* __restrict__ lens, int64_t max_len, T* __restrict__ out,
                                                         int64_t ldo, int heads, float scale) {
    __shared__ float qs[256], ws[64];
    __shared__ int64_t at[64];
    const int lane = threadIdx.x;
    const int64_t r = blockIdx.x / heads;
    const int h = (int)(blockIdx.x - r * heads), g = h / (heads / c.kv_heads);
    const int dh = c.dh, groups = dh >> 5, page = 1 << c.page_shift;
    const int64_t s = seq != nullptr ? seq[r] : r;
    int64_t len = s >= 0 && s < n_seq ? lens[r] : 0;
    len = min(min(len, max_len), width * page);
    for (int e = lane; e < dh; e += 64) qs[e] = load1(q + r * ldq + h * dh + e);
    __syncthreads();
    bool any = false;
    float m = -INFINITY, sum = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t p0 = 0; p0 < len; p0 += 64) {
        const int64_t p = p0 + lane;
        float score = -INFINITY;
        int64_t slot = -1;
        if (p < len) {
            const int32_t pg = table[s * width + (p >> c.page_shift)];
            if (pg >= 0 && ((int64_t)pg << c.page_shift) < c.slots) slot = ((int64_t)pg << c.page_shift) + (p & (page - 1));
        }
        if (slot >= 0) {
            const int64_t row = ((slot >> c.page_shift) * c.kv_heads + g) * page + (slot & (page - 1));
            float a = 0.0f;
            for (int w = 0; w < groups; ++w) {
                const float f = scale_of(c.ks[row * groups + w]);
                for (int e = 0; e < 16; ++e) {
                    const uint32_t b = c.kc[row * (dh >> 1) + w * 16 + e];
                    a = __builtin_fmaf(qs[w * 32 + 2 * e], value_of(b & 15u) * f, a);
                    a = __builtin_fmaf(qs[w * 32 + 2 * e + 1], value_of(b >> 4) * f, a);
                }
            }
            score = a * scale;
        }
        at[lane] = slot;
        const unsigned long long live = __ballot(slot >= 0);
        if (live == 0ull) continue;
        any = true;
        // a NaN score has to reach the result: fmax would drop it
        const unsigned long long nan = __ballot(slot >= 0 && score != score);
        float top = score;
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        const float mn = nan != 0ull ? __builtin_nanf("") : fmaxf(m, top);
        const float w = slot >= 0 && mn != -INFINITY ? __expf(score - mn) : 0.0f;
        const float keep = m == -INFINITY ? 0.0f : __expf(m - mn);
        float total = w;
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
        sum = sum * keep + total;
        m = mn;
        ws[lane] = w;
        __syncthreads();
        for (int u = 0; u < 4; ++u) {
            const int e = lane + 64 * u;
            if (e < dh) {
                acc[u] *= keep;
                for (int j = 0; j < 64; ++j) {
                    if (at[j] < 0) continue;
                    const int64_t ph = (at[j] >> c.page_shift) * c.kv_heads + g;
                    const int tok = (int)(at[j] & (page - 1));
                    const uint32_t b = c.vc[(ph * (dh >> 1) + (e >> 1)) * page + tok];
                    const float f = scale_of(c.vs[(ph * groups + (e >> 5)) * page + tok]);
                    acc[u] = __builtin_fmaf(ws[j], value_of((e & 1) != 0 ? b >> 4 : b & 15u) * f, acc[u]);
                }
            }
        }
        __syncthreads();
    }
    for (int u = 0; u < 4; ++u) {
        const int e = lane + 64 * u;
        if (e < dh) store1(out + r * ldo + h * dh + e, any ? acc[u] / sum : 0.0f);
    }
}

int check_cache(const tst_cache4* c, Cache* o, const char* who) {
    TST_REQUIRE(c != nullptr, TST_ERR_ARG, "%s: null cache", who);
    TST_REQUIRE(tst_dims_ok({c->pages}), TST_ERR_UNSUPPORTED, "%s: a size exceeds 2^31 - 1", who);
    TST_REQUIRE(c->dh == 32 || c->dh == 64 || c->dh == 128 || c->dh == 256, TST_ERR_UNSUPPORTED, "%s: head size %d is not 32, 64, 128 or 256", who, c->dh);
    TST_REQUIRE(c->page == 16 || c->page == 32 || c->page == 64 || c->page == 128, TST_ERR_UNSUPPORTED, "%s: page %d is not 16, 32, 64 or 128", who,
                c->page);
    TST_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 4096 && c->pages >= 0 && c->pages * c->page <= (int64_t)0x7fffffff, TST_ERR_ARG,
                "%s: bad cache sizes (slots are 32-bit)", who);
    TST_REQUIRE(c->pages == 0 || (c->kc && c->ks && c->vc && c->vs), TST_ERR_ARG, "%s: null cache array", who);
    TST_REQUIRE(tst_aligned16(c->kc) && tst_aligned16(c->ks) && tst_aligned16(c->vc) && tst_aligned16(c->vs), TST_ERR_ARG,
                "%s: the cache arrays must be 16-byte aligned", who);
    *o = Cache{c->kc, c->ks, c->vc, c->vs, c->pages * c->page, __builtin_ctz((unsigned)c->page), c->kv_heads, c->dh};
    return TST_OK;
}

template <typename T>
int check_rows(const Cache& c, const T* k, int64_t ldk, const T* v, int64_t ldv, const int32_t* slots, int64_t n, const char* who) {
    TST_REQUIRE(tst_dims_ok({n}), TST_ERR_UNSUPPORTED, "%s: a size exceeds 2^31 - 1", who);
    TST_REQUIRE(n >= 0, TST_ERR_ARG, "%s: negative size", who);
    TST_REQUIRE(n == 0 || (k && v && slots), TST_ERR_ARG, "%s: null pointer", who);
    const int64_t unit = 16 / (int64_t)sizeof(T);
    TST_REQUIRE(ldk % unit == 0 && ldv % unit == 0 && ldk >= (int64_t)c.kv_heads * c.dh && ldv >= (int64_t)c.kv_heads * c.dh, TST_ERR_ARG,
                "%s: leading dimensions must hold kv_heads * dh and be multiples of %d", who, (int)unit);
    TST_REQUIRE(tst_aligned16(k) && tst_aligned16(v), TST_ERR_ARG, "%s: rows must be 16-byte aligned", who);
    return TST_OK;
}

template <typename T>
int cache4_write(const tst_cache4* c, const T* k, int64_t ldk, const T* v, int64_t ldv, const int32_t* slots, int64_t n, void* stream,
                 const char* who) {
    Cache d;
    int rc = check_cache(c, &d, who);
    if (rc == TST_OK) rc = check_rows(d, k, ldk, v, ldv, slots, n, who);
    if (rc != TST_OK || n == 0) return rc;
    const dim3 grid((unsigned)((n + 63) / 64), (unsigned)((d.kv_heads * (d.dh >> 5) + 3) / 4), 2);
    cache4_write_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(d, k, ldk, v, ldv, slots, n);
    return tst_after_launch(who);
}

template <typename T>
int cache4_read(const tst_cache4* c, const int32_t* slots, T* k, int64_t ldk, T* v, int64_t ldv, int64_t n, void* stream, const char* who) {
    Cache d;
    int rc = check_cache(c, &d, who);
    if (rc == TST_OK) rc = check_rows(d, k, ldk, v, ldv, slots, n, who);
    if (rc != TST_OK || n == 0) return rc;
    const dim3 grid((unsigned)((n + 63) / 64), (unsigned)((d.kv_heads * (d.dh >> 5) + 3) / 4), 2);
    cache4_read_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(d, slots, k, ldk, v, ldv, n);
    return tst_after_launch(who);
}

template <typename T>
int attn_cache4(const tst_cache4* c, const T* q, int64_t ldq, const int32_t* table, int64_t width, int64_t n_seq, const int32_t* seq,
                const int32_t* lens, int64_t max_len, T* out, int64_t ldo, int64_t R, int64_t heads, float scale, float* work, int64_t n_work,
                void* stream, const char* who) {
    Cache d;
    int rc = check_cache(c, &d, who);
    if (rc != TST_OK) return rc;
    TST_REQUIRE(tst_dims_ok({R, width, n_seq, max_len, heads}), TST_ERR_UNSUPPORTED, "%s: a size exceeds 2^31 - 1", who);
    TST_REQUIRE(R >= 0 && width >= 0 && n_seq >= 0 && max_len >= 0, TST_ERR_ARG, "%s: negative size", who);
    TST_REQUIRE(heads >= 1 && heads <= 4096 && heads % d.kv_heads == 0, TST_ERR_ARG, "%s: heads must be a multiple of kv_heads", who);
    TST_REQUIRE(R == 0 || (q && out && lens && (n_seq * width == 0 || table)), TST_ERR_ARG, "%s: null pointer", who);
    const int64_t unit = 16 / (int64_t)sizeof(T);
    TST_REQUIRE(ldq % unit == 0 && ldo % unit == 0 && ldq >= heads * d.dh && ldo >= heads * d.dh, TST_ERR_ARG,
                "%s: leading dimensions must hold heads * dh and be multiples of %d", who, (int)unit);
    TST_REQUIRE(tst_aligned16(q) && tst_aligned16(out) && tst_aligned16(work), TST_ERR_ARG, "%s: q, out and work must be 16-byte aligned", who);
    const int64_t need = tst_attn_cache4_work(R, heads, d.kv_heads, d.dh, max_len);
    TST_REQUIRE(need >= 0 && (need == 0 || (work != nullptr && n_work >= need)), TST_ERR_ARG, "%s: work holds %lld floats, %lld are needed", who,
                (long long)n_work, (long long)need);
    if (R == 0) return TST_OK;
    TST_REQUIRE(R * heads <= (int64_t)0x7fffffff, TST_ERR_UNSUPPORTED, "%s: rows * heads exceeds 2^31 - 1", who);
    attn_cache4_kernel<T><<<(unsigned)(R * heads), 64, 0, (hipStream_t)stream>>>(d, q, ldq, table, width, n_seq, seq, lens, max_len, out, ldo,
                                                                                 (int)heads, scale);
    return tst_after_launch(who);
}

}  // namespace

extern "C" int tst_cache4_write_f32(const tst_cache4* c, const float* k, int64_t ldk, const float* v, int64_t ldv, const int32_t* slots,
                                    int64_t n, void* stream) {
    return cache4_write<float>(c, k, ldk, v, ldv, slots, n, stream, "tst_cache4_write_f32");
}
extern "C" int tst_cache4_write_bf16(const tst_cache4* c, const void* k, int64_t ldk, const void* v, int64_t ldv, const int32_t* slots,
                                     int64_t n, void* stream) {
    return cache4_write<__bf16>(c, (const __bf16*)k, ldk, (const __bf16*)v, ldv, slots, n, stream, "tst_cache4_write_bf16");
}
extern "C" int tst_cache4_read_f32(const tst_cache4* c, const int32_t* slots, float* k, int64_t ldk, float* v, int64_t ldv, int64_t n,
                                   void* stream) {
    return cache4_read<float>(c, slots, k, ldk, v, ldv, n, stream, "tst_cache4_read_f32");
}
extern "C" int tst_cache4_read_bf16(const tst_cache4* c, const int32_t* slots, void* k, int64_t ldk, void* v, int64_t ldv, int64_t n,
                                    void* stream) {
    return cache4_read<__bf16>(c, slots, (__bf16*)k, ldk, (__bf16*)v, ldv, n, stream, "tst_cache4_read_bf16");
}

extern "C" int64_t tst_attn_cache4_work(int64_t R, int64_t heads, int64_t kv_heads, int64_t dh, int64_t max_len) {
    (void)R; (void)heads; (void)kv_heads; (void)dh; (void)max_len;
    return 0;
}
extern "C" int tst_attn_cache4_f32(const tst_cache4* c, const float* q, int64_t ldq, const int32_t* table, int64_t width, int64_t n_seq,
                                   const int32_t* seq, const int32_t* lens, int64_t max_len, float* out, int64_t ldo, int64_t R,
                                   int64_t heads, float scale, float* work, int64_t n_work, void* stream) {
    return attn_cache4<float>(c, q, ldq, table, width, n_seq, seq, lens, max_len, out, ldo, R, heads, scale, work, n_work, stream,
                              "tst_attn_cache4_f32");
}
extern "C" int tst_attn_cache4_bf16(const tst_cache4* c, const void* q, int64_t ldq, const int32_t* table, int64_t width, int64_t n_seq,
                                    const int32_t* seq, const int32_t* lens, int64_t max_len, void* out, int64_t ldo, int64_t R,
                                    int64_t heads, float scale, float* work, int64_t n_work, void* stream) {
    return attn_cache4<__bf16>(c, (const __bf16*)q, ldq, table, width, n_seq, seq, lens, max_len, (__bf16*)out, ldo, R, heads, scale, work,
                               n_work, stream, "tst_attn_cache4_bf16");
}
