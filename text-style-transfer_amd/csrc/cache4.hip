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
__device__ __forceinline__ uint32_t scale_to_bits(int s) { return (uint32_t)s << 23; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const bf16x2 v = __builtin_convertvector(f32x2{a, b}, bf16x2);
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float low_f(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_f(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// elements 2 SEL, 2 SEL + 1 of a word of codes; the conversion reads bits 23 .. 30 of the scale only, and gives NaN for scale byte 255
template <int SEL>
__device__ __forceinline__ uint32_t cvt4(uint32_t codes, uint32_t scale_bits) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, __uint_as_float(scale_bits), SEL));
}
template <int SEL>
__device__ __forceinline__ f32x2 cvt4f(uint32_t codes, uint32_t scale_bits) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, __uint_as_float(scale_bits), SEL);
}

// ---- storing and reading back ---------------------------------------------------------------------------------------------------
//
// A workgroup takes 64 rows x 128 elements (4 groups).  Memory sees whole rows of the tile, 16 bytes per lane side by side.  Writing, the 4
// or 8 lanes that hold a group find its scale among them, and only the codes pass through LDS, from where each lane (= row) of a wave
// (= group) takes its 16 bytes; reading, each lane (= row) writes its 32 elements to LDS and rows leave from there (rows padded by 16
// bytes: 16 lanes fall on 16 different 16-byte places).  Key codes leave as 16 bytes per lane.  Value codes lie token by token:
// where the four rows of a lane quad have adjacent slots, the quad transposes its bytes and every lane writes words of four tokens
// (at any byte address), else single bytes.
// Bound by memory: 65521 rows of 8 heads of 128 in fp32 are stored in 142 us (608 MB, 4.3 TB/s) and read back in 114 (5.3 TB/s; a copy of 2
// GB runs at 4.9).  With rows of 512 bytes at a time, column tiles slowest, it was 175 and 135; through LDS in fp32, 168 to store.

constexpr int TILE_ROWS = 64, TILE_COLS = 128;

template <typename T>
struct RowTile {
    static constexpr int ROW_BYTES = TILE_COLS * (int)sizeof(T) + 16;
    static constexpr int CHUNKS = TILE_COLS * (int)sizeof(T) / 16;       // 16-byte pieces per row
};

struct __attribute__((packed, aligned(1))) word_any {
    uint32_t v;
};

// 4 x 4 bytes across the four lanes of a quad: byte b of lane q becomes byte q of lane b
__device__ __forceinline__ uint32_t quad_transpose(uint32_t x, int q) {
    const uint32_t y = (uint32_t)lane_xor_i<1>((int)x);
    x = __builtin_amdgcn_perm(y, x, (q & 1) != 0 ? 0x03070105u : 0x06020400u);
    const uint32_t z = (uint32_t)lane_xor_i<2>((int)x);
    return __builtin_amdgcn_perm(z, x, (q & 2) != 0 ? 0x03020706u : 0x05040100u);
}

// largest of the magnitudes' bits over the LANES lanes that hold a group
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
    x = max(x, (uint32_t)lane_xor_i<1>((int)x));
    x = max(x, (uint32_t)lane_xor_i<2>((int)x));
    if (LANES == 8) x = max(x, (uint32_t)lane_xor_i<4>((int)x));
    return x;
}

template <typename T>
__global__ __launch_bounds__(256) void cache4_write_kernel(Cache c, const T* __restrict__ k, int64_t ldk, const T* __restrict__ v,
                                                           int64_t ldv, const int32_t* __restrict__ slots, int64_t n) {
    constexpr int E = 16 / (int)sizeof(T), CHUNKS = RowTile<T>::CHUNKS, PER = TILE_ROWS * CHUNKS / 256;
    constexpr int CODE_ROW = TILE_COLS / 2 + 16;                           // bytes of codes per row, padded
    __shared__ __attribute__((aligned(16))) unsigned char code_tile[TILE_ROWS * CODE_ROW];
    __shared__ uint32_t scale_tile[TILE_ROWS];                             // the four groups' scale bytes
    // columns fastest, so that the workgroups at work read or write whole rows together
    const int width = c.kv_heads * c.dh, cols = (width + TILE_COLS - 1) / TILE_COLS, col = (int)(blockIdx.x % (unsigned)cols);
    const unsigned rest = blockIdx.x / (unsigned)cols;
    const bool is_v = (rest & 1u) != 0;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t i0 = (int64_t)(rest >> 1) * TILE_ROWS;
    const int rows = (int)min((int64_t)TILE_ROWS, n - i0), col0 = col * TILE_COLS;
    const T* src = is_v ? v + i0 * ldv + col0 : k + i0 * ldk + col0;
    const int64_t ld = is_v ? ldv : ldk;
    uint4 in[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int x = threadIdx.x + 256 * j, r = x / CHUNKS, e = (x % CHUNKS) * E;
        in[j] = *reinterpret_cast<const uint4*>(src + min(r, rows - 1) * ld + (col0 + e < width ? e : 0));    // what is not there goes nowhere
    }
    const int64_t slot = lane < rows ? slots[i0 + lane] : -1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int x = threadIdx.x + 256 * j, r = x / CHUNKS, ch = x % CHUNKS;
        const uint4 u = in[j];
        float y[E];
        if (E == 4) {
            y[0] = __uint_as_float(u.x); y[1] = __uint_as_float(u.y); y[2] = __uint_as_float(u.z); y[3] = __uint_as_float(u.w);
        } else {
            y[0] = low_f(u.x); y[1] = high_f(u.x); y[2] = low_f(u.y); y[3] = high_f(u.y);
            y[E - 4] = low_f(u.z); y[E - 3] = high_f(u.z); y[E - 2] = low_f(u.w); y[E - 1] = high_f(u.w);
        }
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
        const int s = scale_byte(group_max<32 / E>(top));
        const float unit = __uint_as_float(scale_to_bits(s == 255 ? 127 : s));
        // x * 2^-E, rounded to the nearest code, ties to the even one
        uint32_t codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], unit, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[2], y[3], unit, 1);
        if (E == 8) {
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[E - 4], y[E - 3], unit, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[E - 2], y[E - 1], unit, 3);
            *reinterpret_cast<uint32_t*>(code_tile + r * CODE_ROW + 4 * ch) = codes;
        } else {
            *reinterpret_cast<uint16_t*>(code_tile + r * CODE_ROW + 2 * ch) = (uint16_t)codes;
        }
        if ((ch & (32 / E - 1)) == 0) reinterpret_cast<uint8_t*>(scale_tile)[4 * r + ch / (32 / E)] = (uint8_t)s;
    }
    __syncthreads();
    const int groups = c.dh >> 5, hg = col * 4 + w;
    if (hg >= c.kv_heads * groups) return;
    const bool ok = slot >= 0 && slot < c.slots;
    const uint4 mine = *reinterpret_cast<const uint4*>(code_tile + lane * CODE_ROW + 16 * w);
    const uint32_t codes[4] = {mine.x, mine.y, mine.z, mine.w};
    const int s = (int)(scale_tile[lane] >> (8 * w) & 255u);
    const int h = hg / groups, g = hg - h * groups;
    const int page = 1 << c.page_shift, tok = (int)slot & (page - 1);
    const int64_t ph = (ok ? slot >> c.page_shift : 0) * c.kv_heads + h;
    if (!is_v) {
        if (!ok) return;
        *reinterpret_cast<uint4*>(c.kc + ((ph << c.page_shift) + tok) * (c.dh >> 1) + g * 16) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        c.ks[((ph << c.page_shift) + tok) * groups + g] = (uint8_t)s;
        return;
    }
    uint8_t* vc = c.vc + ((ph * (c.dh >> 1) + g * 16) << c.page_shift);
    if (ok) c.vs[((ph * groups + g) << c.page_shift) + tok] = (uint8_t)s;
    // a quad whose slots are s, s + 1, s + 2, s + 3 of one page (a lane's slot is 32-bit)
    const int q = lane & 3, s32 = ok ? (int)slot : -8;
    const int first = __builtin_amdgcn_update_dpp(s32, s32, 0x00, 0xf, 0xf, false);      // the quad's lane 0
    const bool fits = s32 == first + q && first >= 0 && (first & (page - 1)) + 3 < page;
    const unsigned long long bal = __ballot(fits);
    const bool quad = ((bal >> (lane & 60)) & 15ull) == 15ull;
    const int tok0 = first & (page - 1);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const uint32_t t = quad_transpose(codes[d], q);                                  // every lane takes part in the exchange
        if (quad) {
            reinterpret_cast<word_any*>(vc + (((4 * d + q) << c.page_shift) + tok0))->v = t;
        } else if (ok) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vc[((4 * d + e) << c.page_shift) + tok] = (uint8_t)(codes[d] >> (8 * e));
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void cache4_read_kernel(Cache c, const int32_t* __restrict__ slots, T* __restrict__ k, int64_t ldk,
                                                          T* __restrict__ v, int64_t ldv, int64_t n) {
    __shared__ __attribute__((aligned(16))) unsigned char tile[TILE_ROWS * RowTile<T>::ROW_BYTES];
    constexpr int E = 16 / (int)sizeof(T), CHUNKS = RowTile<T>::CHUNKS;
    // columns fastest, so that the workgroups at work read or write whole rows together
    const int width = c.kv_heads * c.dh, cols = (width + TILE_COLS - 1) / TILE_COLS, col = (int)(blockIdx.x % (unsigned)cols);
    const unsigned rest = blockIdx.x / (unsigned)cols;
    const bool is_v = (rest & 1u) != 0;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t i0 = (int64_t)(rest >> 1) * TILE_ROWS;
    const int rows = (int)min((int64_t)TILE_ROWS, n - i0), col0 = col * TILE_COLS;
    const int groups = c.dh >> 5, hg = col * 4 + w;
    if (hg < c.kv_heads * groups) {
        const int64_t slot = lane < rows ? slots[i0 + lane] : -1;
        const bool ok = slot >= 0 && slot < c.slots;
        const int h = hg / groups, g = hg - h * groups;
        const int page = 1 << c.page_shift, tok = (int)slot & (page - 1);
        const int64_t ph = (ok ? slot >> c.page_shift : 0) * c.kv_heads + h;
        uint32_t codes[4] = {0u, 0u, 0u, 0u}, s = 127u;
        if (ok) {
            if (!is_v) {
                const uint4 u = *reinterpret_cast<const uint4*>(c.kc + ((ph << c.page_shift) + tok) * (c.dh >> 1) + g * 16);
                codes[0] = u.x; codes[1] = u.y; codes[2] = u.z; codes[3] = u.w;
                s = c.ks[((ph << c.page_shift) + tok) * groups + g];
            } else {
                const uint8_t* vc = c.vc + ((ph * (c.dh >> 1) + g * 16) << c.page_shift) + tok;
#pragma unroll
                for (int e = 0; e < 16; ++e) codes[e >> 2] |= (uint32_t)vc[e << c.page_shift] << (8 * (e & 3));
                s = c.vs[((ph * groups + g) << c.page_shift) + tok];
            }
        }
        unsigned char* mine = tile + lane * RowTile<T>::ROW_BYTES + w * 32 * (int)sizeof(T);
        const uint32_t f = scale_to_bits((int)s);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if (E == 8) {
                *reinterpret_cast<uint4*>(mine + d * 16) = make_uint4(cvt4<0>(codes[d], f), cvt4<1>(codes[d], f), cvt4<2>(codes[d], f), cvt4<3>(codes[d], f));
            } else {
                const f32x2 a0 = cvt4f<0>(codes[d], f), a1 = cvt4f<1>(codes[d], f), a2 = cvt4f<2>(codes[d], f), a3 = cvt4f<3>(codes[d], f);
                *reinterpret_cast<float4*>(mine + d * 32) = make_float4(a0[0], a0[1], a1[0], a1[1]);
                *reinterpret_cast<float4*>(mine + d * 32 + 16) = make_float4(a2[0], a2[1], a3[0], a3[1]);
            }
        }
    }
    __syncthreads();
    T* dst = is_v ? v + i0 * ldv + col0 : k + i0 * ldk + col0;
    const int64_t ld = is_v ? ldv : ldk;
#pragma unroll
    for (int j = 0; j < TILE_ROWS * CHUNKS / 256; ++j) {
        const int x = threadIdx.x + 256 * j, r = x / CHUNKS, e = (x % CHUNKS) * E;
        if (r < rows && col0 + e < width)
            *reinterpret_cast<uint4*>(dst + r * ld + e) = *reinterpret_cast<const uint4*>(tile + r * RowTile<T>::ROW_BYTES + e * (int)sizeof(T));
    }
}

// ---- attention of single query rows over the cache -----------------------------------------------------------------------------
//
// A wave takes one (row, key head) and walks tiles of 64 tokens; the up to 16 query heads that share the key head are the columns of
// its matrix products, so they cost no further reads.  Per tile, on v_mfma_f32_16x16x32_bf16:
//     S^T [64 tokens x 16 heads] = K [64 x dh] Q^T           four products of 16 tokens
//     O^T [dh x 16 heads]       += V^T [dh x 64] P^T
// Codes become bf16 (exactly) with v_cvt_scalef32_pk_bf16_fp4, which also applies the group's power of two.  The contraction index of
// a product may be permuted if both operands agree, and the layout uses that twice so that nothing ever crosses lanes:
//   - lane quarter j (lane >> 4) loads the dh / 4 adjacent elements j dh / 4 .. of its token's key in one piece (for dh = 128 one 16-byte
//     load and one scale) and calls them its share of the contraction; the query is laid out to match.
//   - row 4 a + i of product u is token 16 a + 4 u + i, so the accumulators of quarter j hold the scores of the 16 adjacent tokens 16 j ..
//     after the four products: exactly the tokens whose value codes quarter j loads as 16 adjacent bytes.
// Running maximum and sum are per lane (one head each); the maximum is shared by the four quarters through two lane exchanges, the sum
// only at the end.  fp32 queries and weights enter as three bf16 pieces (8 + 8 + 8 bits of significand), the codes being exact: fp32
// accuracy at three matrix instructions instead of one.  bf16 queries are one piece and their weights two: what is left of a weight in
// [2^k, 2^(k+1)) is below 2^(k-16), so that the only rounding to bf16 is the output's.  (Weights of one piece, off by up to 2^(k-8): 218.5 us
// instead of 221.5 for the 256 rows below, 36.7 instead of 37.7 for 3 rows of 131001 tokens, but 2.0e-3 instead of 1.7e-3 off the exact outputs.)
//
// Bound by memory: 256 rows of 8 key heads of 128, contexts of up to 8000 tokens (1.09 GB): 221 us, 4.9 TB/s, matrix instructions busy a
// quarter of the time.  Long contexts are split over workgroups (rows x key heads x chunks) and, inside one, over its waves (tile by tile in turn); partial
// (maximum, sum, O) are joined in LDS and by combine_kernel, in a fixed order.

union Frag {
    uint32_t u[4];
    bf16x8 v;
};

__device__ __forceinline__ void store2(float* p, float a, float b) { *reinterpret_cast<f32x2*>(p) = f32x2{a, b}; }
__device__ __forceinline__ void store2(__bf16* p, float a, float b) { *reinterpret_cast<uint32_t*>(p) = pack2(a, b); }

// two floats as NP bf16 pieces each: piece i rounds what the pieces before it left
template <int NP>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&p)[NP]) {
    p[0] = pack2(a, b);
#pragma unroll
    for (int i = 1; i < NP; ++i) {
        a -= low_f(p[i - 1]);
        b -= high_f(p[i - 1]);
        p[i] = pack2(a, b);
    }
}

// byte b of a word of scales, moved to bits 23 .. 30
__device__ __forceinline__ uint32_t scale_bits(uint32_t w, int b) { return b == 0 ? w << 23 : (b == 1 ? w << 15 : (b == 2 ? w << 7 : w >> 1)); }

struct AttendArgs {
    Cache c;
    const void* q;
    int64_t ldq, width, n_seq, max_len, ldo, R;
    const int32_t *table, *seq, *lens;
    void* out;
    float* work;
    int heads, per_kv, head_groups, splits, chunk;
    float scale2;       // |scale| * log2(e), never 0: scores are compared before they are scaled
    int negate;         // the scale is negative: the query changes its sign
};

// The pages of a lane's tokens in the tile at p0: 16 adjacent tokens are in one page; the key rows of a lane are in block (lane & 15) >> 2
// of the tile, its values in block lane >> 4.  Read one tile ahead, so that a tile's loads do not wait for the table.
struct Pages {
    int k, v;
};
__device__ __forceinline__ Pages load_pages(const int32_t* __restrict__ row_table, int page_shift, int p0, int last, int lane) {
    return Pages{row_table[min(p0 + 16 * ((lane & 15) >> 2), last) >> page_shift], row_table[min(p0 + 16 * (lane >> 4), last) >> page_shift]};
}

// key codes and scales of the lane's token of each of the four products
template <int DH>
struct KeyTile {
    uint32_t c[4][DH / 32], s[4];
};
template <int DH>
__device__ __forceinline__ void load_keys(KeyTile<DH>& t, const Cache& c, int pk, int p0, int g, int lane) {
    const int m = lane & 15, j = lane >> 4, page = 1 << c.page_shift;
    pk = (unsigned)pk < (unsigned)(c.slots >> c.page_shift) ? pk : 0;     // a page that does not exist: any page, its tokens count as nothing
    const int64_t row = ((int64_t)pk * c.kv_heads + g) * page + ((p0 + 16 * (m >> 2)) & (page - 1)) + (m & 3);
    const uint8_t* kc = c.kc + row * (DH / 2) + j * (DH / 8);
    const uint8_t* ks = c.ks + row * (DH / 32);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const uint8_t* p = kc + u * 4 * (DH / 2);
        if (DH == 32) t.c[u][0] = *reinterpret_cast<const uint32_t*>(p);
        if (DH == 64) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            t.c[u][0] = x.x; t.c[u][1 % (DH / 32)] = x.y;
        }
        if (DH >= 128) {
#pragma unroll
            for (int q = 0; q < DH / 128; ++q) {
                const uint4 x = reinterpret_cast<const uint4*>(p)[q];
                t.c[u][4 * q % (DH / 32)] = x.x; t.c[u][(4 * q + 1) % (DH / 32)] = x.y;
                t.c[u][(4 * q + 2) % (DH / 32)] = x.z; t.c[u][(4 * q + 3) % (DH / 32)] = x.w;
            }
        }
        const uint8_t* s = ks + u * 4 * (DH / 32);
        if (DH == 256) t.s[u] = *reinterpret_cast<const uint16_t*>(s + 2 * j);
        else t.s[u] = s[DH == 128 ? j : (DH == 64 ? j >> 1 : 0)];
    }
}

// Value codes and scales of the 16 tokens of the lane's quarter.  Row m of the output tiles is spread over the head so that all pieces of a
// lane are of one group of 32 elements (one scale per token): with G groups and 16 / G rows for each, piece b of row m is byte row
// 16 (m / (16 / G)) + (16 / G) b + m % (16 / G), i.e. elements 2 x and 2 x + 1 of that byte row x.
template <int DH>
struct ValueTile {
    uint32_t c[DH / 32][4], s[4];
    int live;           // how many of the tokens count (0 .. 16)
};
template <int DH>
__device__ __forceinline__ int value_row(int m, int b) {
    constexpr int L = 512 / DH;       // 16 / G
    return 16 * (m / L) + L * b + m % L;
}
template <int DH>
__device__ __forceinline__ void load_values(ValueTile<DH>& t, const Cache& c, int pv, int p0, int len, int g, int lane) {
    constexpr int L = 512 / DH;
    const int m = lane & 15, page = 1 << c.page_shift;
    const bool ok = (unsigned)pv < (unsigned)(c.slots >> c.page_shift);
    const int tv = p0 + 16 * (lane >> 4);
    t.live = ok ? max(0, min(16, len - tv)) : 0;
    const int64_t hv = (int64_t)(ok ? pv : 0) * c.kv_heads + g;
    const int iv = tv & (page - 1);
    const uint8_t* vc = c.vc + ((hv * (DH / 2) + value_row<DH>(m, 0)) << c.page_shift) + iv;
    const uint4 y = *reinterpret_cast<const uint4*>(c.vs + ((hv * (DH / 32) + m / L) << c.page_shift) + iv);
    t.s[0] = y.x; t.s[1] = y.y; t.s[2] = y.z; t.s[3] = y.w;
#pragma unroll
    for (int b = 0; b < DH / 32; ++b) {
        const uint4 x = *reinterpret_cast<const uint4*>(vc + ((L * b) << c.page_shift));
        t.c[b][0] = x.x; t.c[b][1] = x.y; t.c[b][2] = x.z; t.c[b][3] = x.w;
    }
}

template <typename T, int DH, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attn_cache4_kernel(AttendArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 3 : 1;     // bf16 pieces of a query element
    constexpr int WP = sizeof(T) == 4 ? 3 : 2;     // and of a weight
    constexpr int KS = DH / 32;                    // steps of a key product
    constexpr int MT = DH / 16;                    // output tiles of 16 elements
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = lane & 15, j = lane >> 4;
    uint32_t id = blockIdx.x;                      // (chunk, row, key head, group of 16 heads)
    const int hg = (int)(id % (uint32_t)a.head_groups);
    id /= (uint32_t)a.head_groups;
    const int g = (int)(id % (uint32_t)a.c.kv_heads);
    id /= (uint32_t)a.c.kv_heads;
    const int64_t r = id % (uint32_t)a.R;
    const int split = (int)(id / (uint32_t)a.R);

    const int64_t s = a.seq != nullptr ? a.seq[r] : r;
    int64_t len = s >= 0 && s < a.n_seq ? a.lens[r] : 0;
    len = max(min(min(len, a.max_len), a.width << a.c.page_shift), (int64_t)0);
    if (split > 0 && (int64_t)split * a.chunk >= len) return;      // the whole workgroup: nothing here, combine_kernel knows
    const int lo = split * a.chunk, hi = (int)min(len, (int64_t)lo + a.chunk);
    const int32_t* row_table = a.table + s * a.width;
    const int col = hg * 16 + n;                   // head of the group this lane's column stands for
    const bool real = col < a.per_kv;
    const int64_t head = (int64_t)g * a.per_kv + col;

    // the query as the B operand: column n, this quarter's dh / 4 elements, 8 per step
    uint32_t q[KS][NP][4];
    {
        const T* qp = (const T*)a.q + r * a.ldq + (real ? head : 0) * DH + j * (DH / 4);
#pragma unroll
        for (int st = 0; st < KS; ++st)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = load1(qp + st * 8 + 2 * e), y = load1(qp + st * 8 + 2 * e + 1);
                if (!real) { x = 0.0f; y = 0.0f; }
                if (a.negate) { x = -x; y = -y; }
                uint32_t p[NP];
                split2<NP>(x, y, p);
#pragma unroll
                for (int i = 0; i < NP; ++i) q[st][i][e] = p[i];
            }
    }
    f32x4 o[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, sum = 0.0f;
    bool any = false;

    int p0 = lo + 64 * w;
    // in flight while a tile is computed: its values during the scores, the next tile's keys during the rest
    KeyTile<DH> keys;
    Pages at, next;
    if (p0 < hi) {
        at = load_pages(row_table, a.c.page_shift, p0, hi - 1, lane);
        next = load_pages(row_table, a.c.page_shift, p0 + 64 * WAVES, hi - 1, lane);
        load_keys<DH>(keys, a.c, at.k, p0, g, lane);
    }
    for (; p0 < hi; p0 += 64 * WAVES) {
        ValueTile<DH> cur;
        load_values<DH>(cur, a.c, at.v, p0, hi, g, lane);
        const unsigned long long full = __ballot(cur.live == 16);
        // scores of this lane's head for the 16 tokens of its quarter: sc[u][i] is token 4 u + i
        f32x4 sc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                const uint32_t word = keys.c[u][st];
                const uint32_t f = DH == 256 && st >= 4 ? keys.s[u] << 15 : keys.s[u] << 23;
                Frag k;
                k.u[0] = cvt4<0>(word, f); k.u[1] = cvt4<1>(word, f); k.u[2] = cvt4<2>(word, f); k.u[3] = cvt4<3>(word, f);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    Frag qq;
                    qq.u[0] = q[st][i][0]; qq.u[1] = q[st][i][1]; qq.u[2] = q[st][i][2]; qq.u[3] = q[st][i][3];
                    sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.v, qq.v, sc[u], 0, 0, 0);
                }
            }
        }
        at = next;
        if (p0 + 64 * WAVES < hi) {
            load_keys<DH>(keys, a.c, at.k, p0 + 64 * WAVES, g, lane);
            next = load_pages(row_table, a.c.page_shift, p0 + 128 * WAVES, hi - 1, lane);
        }
        if (full != ~0ull) {   // the end of the context, or a page that does not exist
            any |= __ballot(cur.live > 0) != 0ull;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int left = min(max(cur.live - 4 * u, 0), 4);
                const uint32_t keep = left == 4 ? 0xffffffffu : (1u << (8 * left)) - 1u;
                cur.s[u] &= keep;
#pragma unroll
                for (int b = 0; b < DH / 32; ++b) cur.c[b][u] &= keep;      // value 0, whatever the page holds there
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[u][i] = i < left ? sc[u][i] : -INFINITY;
            }
        } else {
            any = true;
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[u][i]);
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
        const float base = top == -INFINITY ? 0.0f : top * a.scale2;       // no finite score yet: every weight is exp(-inf) = 0
        if (__ballot(top != m) != 0ull) {
            const float keep = __builtin_amdgcn_exp2f(__builtin_fmaf(m, a.scale2, -base));     // m = -inf: 0
            sum *= keep;
#pragma unroll
            for (int t = 0; t < MT; ++t) o[t] = o[t] * keep;
            m = top;
        }
        // the weights as the B operand: step st holds tokens 8 st .. 8 st + 7 of the quarter
        uint32_t p[2][WP][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][i], a.scale2, -base));
                sum += e[i];
            }
            uint32_t x[WP], y[WP];
            split2<WP>(e[0], e[1], x);
            split2<WP>(e[2], e[3], y);
#pragma unroll
            for (int i = 0; i < WP; ++i) { p[u >> 1][i][2 * (u & 1)] = x[i]; p[u >> 1][i][2 * (u & 1) + 1] = y[i]; }
        }
#pragma unroll
        for (int b = 0; b < DH / 32; ++b) {
            // 16 tokens of the even and of the odd element of this piece's byte row
            Frag even[2], odd[2];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t word = cur.c[b][u], f = cur.s[u];
                const uint32_t t0 = cvt4<0>(word, scale_bits(f, 0)), t1 = cvt4<1>(word, scale_bits(f, 1));
                const uint32_t t2 = cvt4<2>(word, scale_bits(f, 2)), t3 = cvt4<3>(word, scale_bits(f, 3));
                even[u >> 1].u[2 * (u & 1)] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
                even[u >> 1].u[2 * (u & 1) + 1] = __builtin_amdgcn_perm(t3, t2, 0x05040100u);
                odd[u >> 1].u[2 * (u & 1)] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
                odd[u >> 1].u[2 * (u & 1) + 1] = __builtin_amdgcn_perm(t3, t2, 0x07060302u);
            }
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int i = 0; i < WP; ++i) {
                    Frag pp;
                    pp.u[0] = p[st][i][0]; pp.u[1] = p[st][i][1]; pp.u[2] = p[st][i][2]; pp.u[3] = p[st][i][3];
                    o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even[st].v, pp.v, o[2 * b], 0, 0, 0);
                    o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd[st].v, pp.v, o[2 * b + 1], 0, 0, 0);
                }
        }
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (!any) sum = -1.0f;                          // nothing to attend to (a sum of weights is never negative)

    // join the waves: o[2 b + x][i] is element 2 * value_row(4 j + i, b) + x of head n; the maximum becomes one of scaled scores
    m *= a.scale2;
    if (WAVES > 1) {
        __shared__ float red[WAVES][16][2];
        __shared__ float part[WAVES > 1 ? WAVES - 1 : 1][DH][17];
        if (j == 0) { red[w][n][0] = m; red[w][n][1] = sum; }
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top = fmaxf(top, red[i][n][1] < 0.0f ? -INFINITY : red[i][n][0]);
        const float base = top == -INFINITY ? 0.0f : top;
        float total = 0.0f;
        bool some = false;
#pragma unroll
        for (int i = 0; i < WAVES; ++i)
            if (!(red[i][n][1] < 0.0f)) {
                total += red[i][n][1] * __builtin_amdgcn_exp2f(red[i][n][0] - base);
                some = true;
            }
        const float mine = sum < 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - base);
#pragma unroll
        for (int t = 0; t < MT; ++t) o[t] = o[t] * mine;
        if (w > 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[w - 1][4 * MT * j + 4 * t + i][n] = o[t][i];
        }
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < WAVES - 1; ++x) o[t][i] += part[x][4 * MT * j + 4 * t + i][n];
        m = top;
        sum = some ? total : -1.0f;
    }
    if (!real) return;
    if (len <= a.chunk) {                           // the whole row is here
        const float inv = sum < 0.0f ? 0.0f : 1.0f / sum;
        T* op = (T*)a.out + r * a.ldo + head * DH;
#pragma unroll
        for (int b = 0; b < DH / 32; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                store2(op + 2 * value_row<DH>(4 * j + i, b), sum < 0.0f ? 0.0f : o[2 * b][i] * inv, sum < 0.0f ? 0.0f : o[2 * b + 1][i] * inv);
    } else {
        const int64_t at = (r * a.heads + head) * a.splits + split;
        float* ml = a.work + 2 * at;
        float* op = a.work + 2 * a.R * a.heads * a.splits + at * DH;
        if (j == 0) { ml[0] = m; ml[1] = sum; }
#pragma unroll
        for (int b = 0; b < DH / 32; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) store2(op + 2 * value_row<DH>(4 * j + i, b), o[2 * b][i], o[2 * b + 1][i]);
    }
}

// Joins the chunks of the rows that have more than one: one workgroup per (row, head), its eight waves take every eighth chunk, lane = up to
// 4 adjacent elements.
template <typename T, int DH>
__global__ __launch_bounds__(512) void attn_cache4_combine_kernel(AttendArgs a) {
    constexpr int E = DH <= 64 ? 1 : DH / 64;
    __shared__ float part[8][64 * E + 1];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t r = blockIdx.x / (uint32_t)a.heads, head = blockIdx.x - r * a.heads;
    const float* ml = a.work + 2 * (r * a.heads + head) * a.splits;
    const float* op = a.work + 2 * a.R * a.heads * a.splits + (r * a.heads + head) * a.splits * DH;
    // a block of AHEAD chunks: maxima, sums and outputs, requested before the row's length is known (what lies behind it is not used)
    constexpr int AHEAD = 8;
    f32x2 head_ml[AHEAD];
    float piece[AHEAD][E];
    const int el = min(lane * E, DH - E);
    auto request = [&](int i0, int end) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t i = min(i0 + w + 8 * u, end - 1);
            head_ml[u] = *reinterpret_cast<const f32x2*>(ml + 2 * i);
#pragma unroll
            for (int e = 0; e < E; ++e) piece[u][e] = op[i * DH + el + e];
        }
    };
    request(0, a.splits);
    const f32x2 mine = *reinterpret_cast<const f32x2*>(ml + 2 * min(lane, a.splits - 1));
    const int64_t s = a.seq != nullptr ? a.seq[r] : r;
    int64_t len = s >= 0 && s < a.n_seq ? a.lens[r] : 0;
    len = max(min(min(len, a.max_len), a.width << a.c.page_shift), (int64_t)0);
    if (len <= a.chunk) return;
    const int n = (int)((len + a.chunk - 1) / a.chunk);
    float m = -INFINITY;
    bool some = false;
    if (lane < n && !(mine[1] < 0.0f)) { m = mine[0]; some = true; }
    for (int i = lane + 64; i < n; i += 64)
        if (!(ml[2 * i + 1] < 0.0f)) { m = fmaxf(m, ml[2 * i]); some = true; }
    m = wave_max(m);
    some = __ballot(some) != 0ull;
    const float base = m == -INFINITY ? 0.0f : m;
    float acc[E], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int i0 = 0;;) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float si = head_ml[u][1];
            if (i0 + w + 8 * u >= n || si < 0.0f) continue;              // behind the row, or a chunk without tokens
            const float f = __builtin_amdgcn_exp2f(head_ml[u][0] - base);
            sum += si * f;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += piece[u][e] * f;
        }
        if ((i0 += 8 * AHEAD) >= n) break;
        request(i0, n);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) part[w][lane * E + e] = acc[e];
    if (lane == 0) part[w][64 * E] = sum;
    __syncthreads();
    if (w > 0) return;
    sum = 0.0f;
#pragma unroll
    for (int x = 0; x < 8; ++x) sum += part[x][64 * E];
    T* out = (T*)a.out + r * a.ldo + head * DH;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = lane * E + e;
        float total = 0.0f;
#pragma unroll
        for (int x = 0; x < 8; ++x) total += part[x][i];
        if (i < DH) store1(out + i, some ? total / sum : 0.0f);
    }
}

// Positions are counted in 32 bits, up to eight tiles ahead of the last token
constexpr int64_t MOST_TOKENS = 0x7fffffff - 1024;

// How a call is cut: tokens per workgroup (chunk) and how many chunks the longest row may have.  A second launch that joins chunks costs 3 us
// and every chunk a prologue, so rows stay whole where walking one takes no longer: up to 1024 tokens (bf16, 4 key heads of 128, one row of
// 512 tokens: 6.6 us whole, 8.8 cut; 1024 tokens: 8.7 and 8.7; 1536: 10.8 and 8.8), with 128 (row, key head) units up to 2048 (32 rows x 4: 14.3 and
// 15.1), with 256 up to 4096 (64 rows x 4: 26.3 and 30.4; rows of 1 .. 4096 tokens 24.2 and 25.0), with 512 up to 8192 (128 rows x 4, 8192 tokens: 105
// and 110; 256 rows x 8, up to 8000: 220 both).  Longer rows of few units: as many workgroups as run at once, two to a CU (3 rows x 4 key heads,
// 131001 tokens: 37.7 us at 512 workgroups, 40.8 at 768, 37.5 at 1024 with twice the partial results, 44.5 at 384); of many: 1024, so that rows of
// different lengths even out.
void cut(int64_t R, int64_t kv_heads, int64_t head_groups, int64_t max_len, int* chunk, int* splits) {
    const int64_t units = R * kv_heads * head_groups, target = units < 128 ? 512 : 1024;
    const int64_t whole = units < 128 ? 1024 : (units < 256 ? 2048 : (units < 512 ? 4096 : 8192));
    int64_t c = max_len <= whole ? max_len : (max_len * units + target - 1) / target;
    c = (c + 255) / 256 * 256;
    c = c < 256 ? 256 : (c > 8192 ? 8192 : c);
    *chunk = (int)c;
    *splits = max_len > 0 ? (int)((max_len + c - 1) / c) : 1;
}

template <typename T, int DH>
int launch_attend(const AttendArgs& a, hipStream_t st, const char* who) {
    const int64_t groups = a.R * a.c.kv_heads * a.head_groups * a.splits;
    TST_REQUIRE(groups <= (int64_t)0x7fffffff, TST_ERR_UNSUPPORTED, "%s: rows * heads exceeds 2^31 - 1", who);
    if (a.max_len <= 64) attn_cache4_kernel<T, DH, 1><<<(unsigned)groups, 64, 0, st>>>(a);
    else attn_cache4_kernel<T, DH, 4><<<(unsigned)groups, 256, 0, st>>>(a);
    int rc = tst_after_launch(who);
    if (rc == TST_OK && a.splits > 1) {
        attn_cache4_combine_kernel<T, DH><<<(unsigned)(a.R * a.heads), 512, 0, st>>>(a);
        rc = tst_after_launch(who);
    }
    return rc;
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

int tile_grid(const Cache& c, int64_t n, int64_t* grid, const char* who) {
    *grid = (n + TILE_ROWS - 1) / TILE_ROWS * 2 * (((int64_t)c.kv_heads * c.dh + TILE_COLS - 1) / TILE_COLS);
    TST_REQUIRE(*grid <= (int64_t)0x7fffffff, TST_ERR_UNSUPPORTED, "%s: too many rows", who);
    return TST_OK;
}

template <typename T>
int cache4_write(const tst_cache4* c, const T* k, int64_t ldk, const T* v, int64_t ldv, const int32_t* slots, int64_t n, void* stream,
                 const char* who) {
    Cache d;
    int rc = check_cache(c, &d, who);
    if (rc == TST_OK) rc = check_rows(d, k, ldk, v, ldv, slots, n, who);
    if (rc != TST_OK || n == 0) return rc;
    int64_t grid;
    if ((rc = tile_grid(d, n, &grid, who)) != TST_OK) return rc;
    cache4_write_kernel<T><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(d, k, ldk, v, ldv, slots, n);
    return tst_after_launch(who);
}

template <typename T>
int cache4_read(const tst_cache4* c, const int32_t* slots, T* k, int64_t ldk, T* v, int64_t ldv, int64_t n, void* stream, const char* who) {
    Cache d;
    int rc = check_cache(c, &d, who);
    if (rc == TST_OK) rc = check_rows(d, k, ldk, v, ldv, slots, n, who);
    if (rc != TST_OK || n == 0) return rc;
    int64_t grid;
    if ((rc = tile_grid(d, n, &grid, who)) != TST_OK) return rc;
    cache4_read_kernel<T><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(d, slots, k, ldk, v, ldv, n);
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
    TST_REQUIRE(max_len <= MOST_TOKENS, TST_ERR_UNSUPPORTED, "%s: max_len exceeds %lld", who, (long long)MOST_TOKENS);
    TST_REQUIRE(heads >= 1 && heads <= 4096 && heads % d.kv_heads == 0, TST_ERR_ARG, "%s: heads must be a multiple of kv_heads", who);
    TST_REQUIRE(R == 0 || (q && out && lens && (n_seq * width == 0 || table)), TST_ERR_ARG, "%s: null pointer", who);
    const int64_t unit = 16 / (int64_t)sizeof(T);
    TST_REQUIRE(ldq % unit == 0 && ldo % unit == 0 && ldq >= heads * d.dh && ldo >= heads * d.dh, TST_ERR_ARG,
                "%s: leading dimensions must hold heads * dh and be multiples of %d", who, (int)unit);
    TST_REQUIRE(tst_aligned16(q) && tst_aligned16(out) && tst_aligned16(work), TST_ERR_ARG, "%s: q, out and work must be 16-byte aligned", who);
    int chunk, splits;
    cut(R, d.kv_heads, (heads / d.kv_heads + 15) / 16, max_len, &chunk, &splits);
    const int64_t need = splits > 1 ? R * heads * splits * (d.dh + 2) : 0;
    TST_REQUIRE(need == 0 || (work != nullptr && n_work >= need), TST_ERR_ARG, "%s: work holds %lld floats, %lld are needed", who,
                (long long)n_work, (long long)need);
    TST_REQUIRE(scale - scale == 0.0f, TST_ERR_ARG, "%s: scale is not finite", who);
    if (R == 0) return TST_OK;
    TST_REQUIRE(R * heads <= (int64_t)0x7fffffff, TST_ERR_UNSUPPORTED, "%s: rows * heads exceeds 2^31 - 1", who);
    if (d.slots == 0 || width == 0 || n_seq == 0) max_len = 0;     // nothing can be attended to: zeros
    AttendArgs a{d, q, ldq, width, n_seq, max_len, ldo, R, table, seq, lens, out, work, (int)heads, (int)(heads / d.kv_heads),
                 (int)((heads / d.kv_heads + 15) / 16), 1, 0, fmaxf(fabsf(scale) * 1.44269504088896341f, 1e-37f), scale < 0.0f ? 1 : 0};
    cut(R, d.kv_heads, a.head_groups, max_len, &a.chunk, &a.splits);
    hipStream_t st = (hipStream_t)stream;
    if (d.dh == 32) return launch_attend<T, 32>(a, st, who);
    if (d.dh == 64) return launch_attend<T, 64>(a, st, who);
    if (d.dh == 128) return launch_attend<T, 128>(a, st, who);
    return launch_attend<T, 256>(a, st, who);
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
    if (R < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || dh < 1 || max_len < 0 || max_len > MOST_TOKENS || !tst_dims_ok({R, heads, dh}) || !tst_dims_ok({R * heads})) return -1;
    if (max_len <= 1024) return 0;                   // whole rows, however few
    // The most partial results of any r <= R rows: chunks of at least max_len * units / target tokens are at most target / units + 1 of a row,
    // and chunks of 8192, where that is more, ceil(max_len / 8192).
    const int64_t per_row = kv_heads * ((heads / kv_heads + 15) / 16), most = R * ((max_len + 8191) / 8192), even = (1024 + per_row - 1) / per_row + R;
    const int64_t parts = R * ((max_len + 255) / 256), cut_parts = most > even ? most : even;
    return (parts < cut_parts ? parts : cut_parts) * heads * (dh + 2);
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
