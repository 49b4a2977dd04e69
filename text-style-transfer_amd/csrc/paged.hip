// Page tables and slot maps of a paged cache, built on the GPU from the lengths of the sequences (integers only).
//
// A launch is split over groups of adjacent sequences (blockIdx.x) and, within a group, over its tokens (blockIdx.y).  Every
// workgroup first adds up the tokens and pages of ALL sequences in front of its group: at most a few thousand lengths out of
// the L2, cheaper than a second launch that would wait for a scan.  Then it scans its own group in LDS and writes table rows
// and token entries; a lane takes four adjacent tokens, one search and three 16-byte stores.
// 8192 sequences, 2.1 M tokens (27 MB): 10.8 us, of which the sums in front of the groups are 4; 18.8 with one token per lane.  48
// sequences: 4.5 us, a launch and the chain of loads lengths -> offsets -> pages.
#include "tst_common.h"

namespace {

constexpr int MAX_GROUP = 64;   // sequences per workgroup: one lane each in the group's scan

struct PlanArgs {
    const int32_t *lens, *room, *pages;
    int32_t *table, *cu, *slots, *pos, *seq, *used;
    int64_t B, n_pages, N, width;
    int page_shift, group;
    int aligned_in, aligned_out;    // lens and room / slots, pos and seq start at 16-byte boundaries
};

// pages of a sequence, in 32 bits: len + room may pass 2^31
__device__ __forceinline__ int32_t need_of(const PlanArgs& a, int len, int room) {
    const uint32_t n = (uint32_t)max(len, 0), r = (uint32_t)max(room, 0), m = (1u << a.page_shift) - 1u;
    const uint32_t need = (n >> a.page_shift) + (r >> a.page_shift) + (((n & m) + (r & m) + m) >> a.page_shift);
    return (int32_t)min(need, (uint32_t)a.width);
}
__device__ __forceinline__ int32_t clip31(int64_t v) { return v > 0x7fffffff ? 0x7fffffff : (int32_t)v; }

template <int NT>
__global__ __launch_bounds__(NT) void page_plan_kernel(PlanArgs a) {
    __shared__ int64_t part[2][NT / 64];
    __shared__ int tok0[MAX_GROUP + 1], page0[MAX_GROUP + 1];      // within the group; entries behind its last sequence hold the totals
    const int t = threadIdx.x, lane = t & 63;
    const int64_t b0 = (int64_t)blockIdx.x * a.group;
    const int nb = (int)min((int64_t)a.group, a.B - b0);
    int64_t st = 0, sp = 0;
    int64_t b = 0;
    if (a.aligned_in) {
        const int64_t quads = b0 >> 2;
#pragma unroll 4
        for (int64_t i = t; i < quads; i += NT) {
            const int4 n = reinterpret_cast<const int4*>(a.lens)[i];
            const int4 m = a.room != nullptr ? reinterpret_cast<const int4*>(a.room)[i] : make_int4(0, 0, 0, 0);
            st += (int64_t)max(n.x, 0) + max(n.y, 0) + max(n.z, 0) + max(n.w, 0);
            sp += (int64_t)need_of(a, n.x, m.x) + need_of(a, n.y, m.y) + need_of(a, n.z, m.z) + need_of(a, n.w, m.w);
        }
        b = quads << 2;
    }
    for (b += t; b < b0; b += NT) {
        const int n = a.lens[b];
        st += max(n, 0);
        sp += need_of(a, n, a.room != nullptr ? a.room[b] : 0);
    }
    for (int off = 32; off > 0; off >>= 1) {
        st += __shfl_xor(st, off, 64);
        sp += __shfl_xor(sp, off, 64);
    }
    if (lane == 0) { part[0][t >> 6] = st; part[1][t >> 6] = sp; }
    if (t < 64) {   // scan of the group: one sequence per lane
        int64_t n = 0, p = 0;
        if (lane < nb) {
            const int len = a.lens[b0 + lane];
            n = max(len, 0);
            p = need_of(a, len, a.room != nullptr ? a.room[b0 + lane] : 0);
        }
        int64_t in = n, ip = p;
        for (int off = 1; off < 64; off <<= 1) {
            const int64_t un = __shfl_up(in, off, 64), up = __shfl_up(ip, off, 64);
            if (lane >= off) { in += un; ip += up; }
        }
        tok0[lane] = clip31(in - n);
        page0[lane] = clip31(ip - p);
        if (lane == 63) { tok0[64] = clip31(in); page0[64] = clip31(ip); }
    }
    __syncthreads();
    int64_t t_base = 0, p_base = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) { t_base += part[0][i]; p_base += part[1][i]; }
    if (blockIdx.y == 0) {
        if (t < nb) a.cu[b0 + t] = clip31(t_base + tok0[t]);
        if (t == 0 && b0 + nb == a.B) {
            a.cu[a.B] = clip31(t_base + tok0[MAX_GROUP]);
            a.used[0] = clip31(p_base + page0[MAX_GROUP]);
        }
    }
    // table rows of the group, entry by entry
    const int64_t cells = (int64_t)nb * a.width;
    for (int64_t i = (int64_t)blockIdx.y * NT + t; i < cells; i += (int64_t)gridDim.y * NT) {
        const int s = cells <= 0x7fffffff ? (int)((uint32_t)i / (uint32_t)a.width) : (int)(i / a.width);
        const int64_t j = i - (int64_t)s * a.width, at = p_base + page0[s] + j;
        a.table[(b0 + s) * a.width + j] = (page0[s] + j < page0[s + 1] && at < a.n_pages) ? a.pages[at] : -1;
    }
    // tokens of the group: lane quads of adjacent tokens, at multiples of four of the packed index
    const int mask = (1 << a.page_shift) - 1;
    const int64_t lo = t_base, hi = min(t_base + tok0[MAX_GROUP], a.N);
    for (int64_t q = (lo >> 2) + (int64_t)blockIdx.y * NT + t; 4 * q < hi; q += (int64_t)gridDim.y * NT) {
        const int64_t i0 = max(4 * q, lo);
        const int r0 = (int)(i0 - lo);
        int s = 0;
        for (int step = MAX_GROUP / 2; step > 0; step >>= 1)   // the last sequence that starts at or before the token: it holds it
            if (s + step < nb && tok0[s + step] <= r0) s += step;
        int start = tok0[s], end = tok0[s + 1], pg0 = page0[s], pg1 = page0[s + 1], have = -1, pg = -1;
        int v_slot[4], v_pos[4], v_seq[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t i = 4 * q + e;
            v_slot[e] = -1; v_pos[e] = 0; v_seq[e] = 0;
            if (i < lo || i >= hi) continue;
            const int r = (int)(i - lo);
            while (r >= end) {                                 // empty sequences are skipped
                ++s;
                start = end; end = tok0[s + 1];
                pg0 = page0[s]; pg1 = page0[s + 1];
                have = -1;
            }
            const int p = r - start, j = p >> a.page_shift;
            if (j != have) {
                const int64_t at = p_base + pg0 + j;
                pg = (pg0 + j < pg1 && at < a.n_pages) ? a.pages[at] : -1;
                have = j;
            }
            v_slot[e] = pg >= 0 ? clip31(((int64_t)pg << a.page_shift) + (p & mask)) : -1;
            v_pos[e] = p;
            v_seq[e] = (int)b0 + s;
        }
        if (a.aligned_out && 4 * q >= lo && 4 * q + 4 <= hi) {
            reinterpret_cast<int4*>(a.slots)[q] = make_int4(v_slot[0], v_slot[1], v_slot[2], v_slot[3]);
            reinterpret_cast<int4*>(a.pos)[q] = make_int4(v_pos[0], v_pos[1], v_pos[2], v_pos[3]);
            reinterpret_cast<int4*>(a.seq)[q] = make_int4(v_seq[0], v_seq[1], v_seq[2], v_seq[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t i = 4 * q + e;
                if (i < lo || i >= hi) continue;
                a.slots[i] = v_slot[e];
                a.pos[i] = v_pos[e];
                a.seq[i] = v_seq[e];
            }
        }
    }
}

__global__ __launch_bounds__(256) void page_step_kernel(const int32_t* __restrict__ base, const int32_t* __restrict__ sent, int64_t t,
                                                        const int32_t* __restrict__ table, int64_t width, int64_t n_seq, int page_shift,
                                                        int32_t* __restrict__ slots, int32_t* __restrict__ pos, int32_t* __restrict__ lens,
                                                        int64_t R, int64_t limit) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= R) return;
    const int64_t s = sent != nullptr ? sent[r] : r;
    int32_t slot = -1, ps = 0, len = 0;
    const int64_t p = s >= 0 && s < n_seq ? (int64_t)max(base[s], 0) + t : limit;
    if (p < limit) {
        ps = clip31(p);
        len = clip31(p + 1);
        const int64_t j = p >> page_shift;
        if (j < width) {
            const int32_t pg = table[s * width + j];
            if (pg >= 0) slot = clip31(((int64_t)pg << page_shift) + (p & ((1 << page_shift) - 1)));
        }
    }
    slots[r] = slot;
    pos[r] = ps;
    lens[r] = len;
}

int page_shift_of(int64_t page) {
    for (int s = 3; s <= 10; ++s)
        if (page == (int64_t)1 << s) return s;
    return -1;
}

}  // namespace

extern "C" int tst_page_plan(const int32_t* lens, const int32_t* room, int64_t B, const int32_t* pages, int64_t n_pages, int64_t page,
                             int32_t* table, int64_t width, int32_t* cu, int32_t* slots, int32_t* pos, int32_t* seq, int64_t N,
                             int32_t* used, void* stream) {
    TST_REQUIRE(tst_dims_ok({B, n_pages, width, N}), TST_ERR_UNSUPPORTED, "tst_page_plan: a size exceeds 2^31 - 1");
    TST_REQUIRE(B >= 0 && n_pages >= 0 && width >= 0 && N >= 0, TST_ERR_ARG, "tst_page_plan: negative size");
    const int shift = page_shift_of(page);
    TST_REQUIRE(shift >= 0, TST_ERR_ARG, "tst_page_plan: page must be a power of two in 8 .. 1024");
    TST_REQUIRE(cu && used && (B == 0 || lens) && (n_pages == 0 || pages) && (B * width == 0 || table) && (N == 0 || (slots && pos && seq)),
                TST_ERR_ARG, "tst_page_plan: null pointer");
    // groups: small enough to spread the writes over the chip, large enough that the sums in front of the groups stay cheap
    int64_t group = 1;
    while (group < MAX_GROUP && group * 512 < B) group *= 2;
    const int64_t groups = B > 0 ? (B + group - 1) / group : 1;
    // many sequences: larger workgroups, fewer of which read the lengths (8192 sequences: 1024 threads 10.8 us, 512 11.6, 256 12.2; 48: 4.9, 4.6
    // and 4.5)
    const int64_t nt = B > 1024 ? 1024 : 256, share = B > 1024 ? 8192 : 4096;            // threads; tokens and table cells of a workgroup
    int64_t slices = (N + B * width + groups * share - 1) / (groups * share);
    slices = slices < 1 ? 1 : (slices > 1024 ? 1024 : slices);
    const PlanArgs a{lens, room, pages, table, cu, slots, pos, seq, used, B, n_pages, N, width, shift, (int)group,
                     tst_aligned16(lens) && tst_aligned16(room), tst_aligned16(slots) && tst_aligned16(pos) && tst_aligned16(seq)};
    const dim3 grid((unsigned)groups, (unsigned)slices);
    if (nt == 1024) page_plan_kernel<1024><<<grid, 1024, 0, (hipStream_t)stream>>>(a);
    else page_plan_kernel<256><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    return tst_after_launch("tst_page_plan");
}

// the rows' positions are below `limit`; others are treated like rows of no sequence
int tst_page_step_within(const int32_t* base, const int32_t* sent, int64_t t, const int32_t* table, int64_t width, int64_t n_seq, int64_t page,
                         int32_t* slots, int32_t* pos, int32_t* lens, int64_t R, int64_t limit, void* stream) {
    TST_REQUIRE(tst_dims_ok({t, width, n_seq, R}), TST_ERR_UNSUPPORTED, "tst_page_step: a size exceeds 2^31 - 1");
    TST_REQUIRE(t >= 0 && width >= 0 && n_seq >= 0 && R >= 0, TST_ERR_ARG, "tst_page_step: negative size");
    const int shift = page_shift_of(page);
    TST_REQUIRE(shift >= 0, TST_ERR_ARG, "tst_page_step: page must be a power of two in 8 .. 1024");
    TST_REQUIRE(R == 0 || (slots && pos && lens && (n_seq == 0 || (base && (width == 0 || table)))), TST_ERR_ARG, "tst_page_step: null pointer");
    if (R == 0) return TST_OK;
    page_step_kernel<<<(unsigned)((R + 255) / 256), 256, 0, (hipStream_t)stream>>>(base, sent, t, table, width, n_seq, shift, slots, pos, lens, R, limit);
    return tst_after_launch("tst_page_step");
}

extern "C" int tst_page_step(const int32_t* base, const int32_t* sent, int64_t t, const int32_t* table, int64_t width, int64_t n_seq,
                             int64_t page, int32_t* slots, int32_t* pos, int32_t* lens, int64_t R, void* stream) {
    return tst_page_step_within(base, sent, t, table, width, n_seq, page, slots, pos, lens, R, INT64_MAX, stream);
}
