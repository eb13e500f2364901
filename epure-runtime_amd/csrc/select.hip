// Bounds of a paged cache's keys, and the pages of a context that matter most
// to a token by them (include/epure_paged.h).  Attention over those pages is
// attend_kernel.h.
//
//   lo_d, hi_d = least and largest key value of column d over a page's rows
//   score(page) = sum_d hi_d sum_g max(q_gd, 0) + lo_d sum_g min(q_gd, 0)
//
// over the query heads g that share the cache head: every product q_gd k_d of a
// row of the page is at most its term, so the group's scores of no position
// there sum to more.  The heads enter as two vectors, so the work does not
// grow with them: 2 D multiply-adds a page.
//
// The choice is a whole number, so the scores are sums in 64 bits: the
// products of 16-bit values are exact there, and pages next to the border
// do not change places with the order of a sum, as they would in 32 bits.
//
// Scores are bound by the bytes of the bounds: 8 sequences of 2048 pages on 8
// heads of 128 (bf16, 67 MB) take 17 us and the choice of 64 of them 8, a chain
// of steps over LDS.  Up to kFewPages pages a row one workgroup does both in one
// launch (44 pages on 8 heads: 7.4 us; 60 tokens of up to 282 pages on 4: 12.8).
// The bounds of 64 appended tokens take 6.1 us, a chain of loads, and those of
// 2 x 4096 (8 heads, pages of 64) 12.0, beside 14.4 for the rows themselves.
#include "ep_common.h"
#include "ep_internal.h"
#include "ep_paged.h"

#include <algorithm>
#include <type_traits>

namespace ep {
namespace {

constexpr int kGroupTokens = 64;    // tokens that a wave looks over at a time for the bounds
constexpr int kRowChunks = 64;      // workgroups that share a row of tokens for them, at most
constexpr int kChunkPages = 128;    // pages a workgroup scores
constexpr int kHeldKeys = 4096;     // scores that the choice keeps in LDS (32 KiB)
constexpr int kFewPages = 512;      // of a table whose rows one workgroup each scores and chooses from

struct BoundsArgs {
    PagedTokens tok;
    PagedCache c;
    void *bounds;
    int64_t limit;           // positions from here on store nothing
    uint32_t first_wg, chunks, each;     // workgroups a sequence, of `each` groups of tokens
    uint32_t heads, head_groups;         // that a workgroup takes one after the other; workgroups that share all
};

// Eight adjacent values of a cache row as f32.
template <int CODE>
EP_DEV void row_values(const PagedCache &c, int64_t row, int d, float *v)
{
    if constexpr (CODE == EP_I8 || CODE == EP_E4M3) {
        const float s = c.k_scale[row];
        uint32_t w[2];
        __builtin_memcpy(w, __builtin_assume_aligned((const uint8_t *)c.k + row * c.D + d, 8), 8);
        decode4(w[0], CODE, v);
        decode4(w[1], CODE, v + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] *= s;
    } else {
        uint16_t r[8];
        __builtin_memcpy(r, __builtin_assume_aligned((const uint16_t *)c.k + row * c.D + d, 16), 16);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = CODE == EP_F16 ? (float)f16_from_bits(r[i]) : bf16_to_f32(r[i]);
    }
}

// A NaN stays: a page that holds one is not to be passed over.
EP_DEV float least(float a, float b) { return b < a || b != b ? b : a; }
EP_DEV float largest(float a, float b) { return b > a || b != b ? b : a; }

// The next lane's value (the last lane's: anything).
EP_DEV int64_t next_lane(int64_t v)
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, 0x130, 0xf, 0xf, false);     // wave_shl:1
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), 0x130, 0xf, 0xf, false);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// One workgroup looks over `each` times 64 tokens of a sequence, for one cache head
// or a few.
// Of the tokens on one page the one at the largest position (of two there, the
// later in the call) rebuilds the page's bounds from its rows up to that position:
// what the page held before the call counts as the new rows do, nothing that it
// held for an earlier sequence does, and it does not matter how often it is done.
// Where positions ascend (padded at either end, all below the limit) that token is
// the one whose successor lies elsewhere; in any other order the whole row is
// searched for a later one, once a page.  A page may be in other sequences' tables
// too, at the same place: the rows of those are searched as well (a load a sequence
// finds that there are none, as a rule; 16 x 4096 tokens in chunks over one table
// of pages of 64, 8 heads of 128, append included: 334 us, of which 227 are that
// search).
// WAVES waves share a page: all four, or one; 0: all four, and rows are of one
// token (code for several, fetched cold, took 0.7 us more).
template <int CODE, int WAVES>
__global__ void __launch_bounds__(256) bounds_kernel(BoundsArgs a)
{
    constexpr bool ONE = WAVES == 0;
    constexpr int TEAMS = WAVES == 1 ? 4 : 1, TEAM = 256 / TEAMS, kOrder = WAVES == 1 ? 16 : 8;
    __shared__ float s_lo[256 * 8], s_hi[256 * 8];
    const uint32_t at = a.first_wg + blockIdx.x, H = a.c.heads;
    const uint32_t part = at / a.head_groups, h0 = (at - part * a.head_groups) * a.heads, h1 = min(h0 + a.heads, H);
    const uint32_t b = ONE ? part : part / a.chunks, chunk = part - b * a.chunks;
    const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM, lane = tid & 63, D = a.c.D;
    const int64_t *pos = a.tok.pos + (int64_t)b * a.tok.pos_sb;
    auto stored = [&](int64_t p) { return p < a.limit ? p : -1; };
    const int64_t ps = a.tok.pos_ss, s_begin = (int64_t)chunk * a.each * kGroupTokens;
    const int64_t s_end = s_begin + a.each * kGroupTokens < a.tok.S ? s_begin + a.each * kGroupTokens : a.tok.S;
    bool ascend = true;
    if constexpr (!ONE) {
        int wrong = 0, begins = 0;
        for (int64_t t0 = threadIdx.x; t0 < a.tok.S; t0 += kOrder * 256) {
            int64_t o[kOrder], after[kOrder];
#pragma unroll
            for (int i = 0; i < kOrder; ++i) {      // all in flight; past the end the first again
                const int64_t t = t0 + 256 * i < a.tok.S ? t0 + 256 * i : t0;
                o[i] = pos[t * ps];
                after[i] = -1;
                if (lane == 63 && t + 1 < a.tok.S)
                    after[i] = pos[(t + 1) * ps];
            }
#pragma unroll
            for (int i = 0; i < kOrder; ++i) {
                const int64_t next = next_lane(o[i]), t = t0 + 256 * i < a.tok.S ? t0 + 256 * i : t0;
                after[i] = lane == 63 ? after[i] : t + 1 < a.tok.S ? next : -1;
                wrong |= (after[i] >= 0 && after[i] <= o[i]) || o[i] >= a.limit;
                begins += o[i] < 0 && after[i] >= 0 && t0 + 256 * i < a.tok.S;
            }
        }
        // behind a token that is none they may begin once, where the first is none
        const int threads = __syncthreads_count(begins);
        ascend = !__syncthreads_or(wrong || begins > 1) && threads <= (pos[0] < 0);
    }
    // LDS of a team of one wave: its own accesses stay in order
    auto team_sync = [&]() {
        if constexpr (TEAMS == 1)
            __syncthreads();
        else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
        }
    };
    auto team_any = [&](int x) {
        if constexpr (TEAMS == 1)
            return __syncthreads_or(x);
        else
            return __any(x);
    };
    // This thread's share of a look for a token between position `mine` and `top`
    // among the positions o of a sequence; at `mine`: behind token `who`.
    auto later_in = [&](const int64_t *o, int64_t mine, int64_t top, int64_t who) {
        int later = 0;
        for (int64_t t0 = tid; t0 < a.tok.S; t0 += 8 * TEAM) {
            int64_t p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)      // eight loads in flight; past the end the first again
                p[i] = o[(t0 + TEAM * i < a.tok.S ? t0 + TEAM * i : t0) * ps];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t t = t0 + TEAM * i < a.tok.S ? t0 + TEAM * i : t0;
                const uint64_t ahead = p[i] - mine;
                later |= ahead < (uint64_t)(top - mine) && (ahead || t > who);
            }
        }
        return later;
    };
    float *const t_lo = s_lo + 8 * TEAM * team, *const t_hi = s_hi + 8 * TEAM * team;
    const int lanes = D / 8, group = tid / lanes, u = tid - group * lanes, groups = TEAM / lanes;
    for (int64_t s0 = s_begin + kGroupTokens * team; s0 < s_end; s0 += kGroupTokens * TEAMS) {
        const int64_t s = s0 + lane;
        const int64_t p = stored(ONE ? pos[0] : s < a.tok.S ? pos[s * ps] : -1);
        const int64_t after = stored(!ONE && s + 1 < a.tok.S ? pos[(s + 1) * ps] : -1);
        const int64_t index = p >> a.c.page_shift;
        int32_t id = -1;
        if (p >= 0 && index < a.tok.width)
            id = a.tok.table[b * a.tok.table_stride + index];
        // not the last one there: where positions ascend, any on the page that follows; else
        // the next token on the next row
        const bool inner = after >> a.c.page_shift == index && (ascend ? after >= 0 : after == p + 1);
        uint64_t left = __ballot(id >= 0 && id < a.c.n_pages && !inner);
        for (; left; left &= left - 1) {
            const int l = ONE ? 0 : __builtin_ctzll(left);
            const int64_t mine = __shfl(p, l, 64), page = mine >> a.c.page_shift, who = s0 + l;
            const int32_t here = __shfl(id, l, 64);
            const int64_t end = (page + 1) << a.c.page_shift, top = end < a.limit ? end : a.limit;
            int later = 0;
            if constexpr (ONE)       // the loads do not wait for `here`
                for (int64_t o = tid; o < a.tok.B; o += 256) {
                    const int32_t there = a.tok.table[o * a.tok.table_stride + page];
                    const int64_t q = a.tok.pos[o * a.tok.pos_sb];
                    later |= there == here && q > mine && q < top;
                }
            else if (!ascend || a.tok.B > 1) {
                for (int64_t o0 = 0; o0 < a.tok.B; o0 += 64) {
                    const int64_t o = o0 + lane;
                    bool have = o < a.tok.B;
                    if (have)
                        have = o == b ? !ascend : a.tok.table[o * a.tok.table_stride + page] == here;
                    for (uint64_t rows = __ballot(have); rows; rows &= rows - 1) {
                        const int64_t r = o0 + __builtin_ctzll(rows);
                        later |= later_in(a.tok.pos + r * a.tok.pos_sb, mine, top, r == b ? who : a.tok.S);
                    }
                }
                if (team_any(later))
                    continue;
            }
            const int rows = (int)(mine & (a.c.page - 1)) + 1;
            for (uint32_t h = h0; h < h1; ++h) {
                const int64_t row0 = ((int64_t)here * H + h) * a.c.page;
                float lo[8], hi[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    lo[i] = INFINITY;
                    hi[i] = -INFINITY;
                }
                if (group < groups)
                    for (int r = group; r < rows; r += 4 * groups) {
                        float v[4][8];
#pragma unroll
                        for (int k = 0; k < 4; ++k)      // four rows in flight; past the end the last again
                            row_values<CODE>(a.c, row0 + min(r + k * groups, rows - 1), 8 * u, v[k]);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                lo[i] = least(lo[i], v[k][i]);
                                hi[i] = largest(hi[i], v[k][i]);
                            }
                    }
                if (ONE && h == h0) {
                    if (a.tok.B > 1 && team_any(later))
                        return;
                } else
                    team_sync();     // the buffers' last readers are done
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    t_lo[8 * tid + i] = lo[i];      // [group][D], as 8 (group lanes + u) + i = group D + 8 u + i
                    t_hi[8 * tid + i] = hi[i];
                }
                team_sync();
                const int64_t out = ((int64_t)here * H + h) * 2 * D;
                for (int e = tid; e < 2 * D; e += TEAM) {
                    const bool top = e >= D;
                    const int d = top ? e - D : e;
                    float x = top ? t_hi[d] : t_lo[d];
                    for (int k = 1; k < groups; ++k)
                        x = top ? largest(x, t_hi[k * D + d]) : least(x, t_lo[k * D + d]);
                    if constexpr (CODE == EP_F16)
                        ((f16_t *)a.bounds)[out + e] = (f16_t)x;
                    else if constexpr (CODE == EP_BF16)
                        ((uint16_t *)a.bounds)[out + e] = f32_to_bf16(x);
                    else
                        ((float *)a.bounds)[out + e] = x;
                }
            }
            if (ONE)
                return;
        }
        if (ONE)
            return;
    }
}

struct SelectArgs {
    const void *q;
    int64_t q_sb, q_ss, q_sh;
    int q_dtype, G;
    PagedTokens tok;
    PagedCache c;
    const void *bounds;
    uint64_t *keys;          // [rows][width]
    int32_t *blocks;         // [rows][take]
    uint32_t first_wg, chunks;
    int take, lanes;         // lanes: that hold a page's D columns, eight each, a power of two
};

// Row r: a token's cache head, and the page that the token lies on (-1: none).
struct SelectRow {
    uint32_t token, h;
    int64_t b, s, own;
};
EP_DEV SelectRow select_row(const SelectArgs &a, uint32_t r)
{
    SelectRow o;
    o.token = r / (uint32_t)a.c.heads;
    o.h = r - o.token * a.c.heads;
    o.b = o.token / (uint32_t)a.tok.S;
    o.s = o.token - o.b * a.tok.S;
    const int64_t p = a.tok.pos[o.b * a.tok.pos_sb + o.s * a.tok.pos_ss], page = p >> a.c.page_shift;
    o.own = p < 0 || page >= a.tok.width ? -1 : page;
    return o;
}

template <int CTRL>
EP_DEV double dpp_f64(double v)
{
    const uint64_t b = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)b, CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
    return __longlong_as_double(((uint64_t)hi << 32) | lo);
}

// Sum over `lanes` adjacent lanes (a power of two, at most 32).
EP_DEV double lanes_sum(double v, int lanes)
{
    if (lanes > 1)
        v += dpp_f64<0xb1>(v);      // quad_perm [1,0,3,2]
    if (lanes > 2)
        v += dpp_f64<0x4e>(v);      // quad_perm [2,3,0,1]
    if (lanes > 4)
        v += dpp_f64<0x141>(v);     // row_half_mirror
    if (lanes > 8)
        v += dpp_f64<0x140>(v);     // row_mirror
    if (lanes > 16)
        v += __shfl_xor(v, 16, 64);
    return v;
}

// Scores as integers of the same order: a NaN above all (a page that holds
// one, or that the pool lacks, is not to be passed over).
EP_DEV uint64_t order_key(double v)
{
    const uint64_t b = __double_as_longlong(v + 0.0);       // one zero
    if (v != v)
        return ~0ull;
    return b >> 63 ? ~b : b | 1ull << 63;
}

// Eight bounds of either kind, one of them low or high.
template <bool WIDE>
struct Bounds8 {
    u32x4_t w[WIDE ? 2 : 1];
    EP_DEV void load(const void *p, int64_t at)
    {
        const u32x4_t *src = (const u32x4_t *)((const char *)p + at * (WIDE ? 4 : 2));
        w[0] = src[0];
        if constexpr (WIDE)
            w[1] = src[1];
    }
    EP_DEV float at(int i, bool f16) const
    {
        if constexpr (WIDE)
            return __uint_as_float(w[i / 4][i % 4]);
        const uint16_t b = (uint16_t)(w[0][i / 2] >> (16 * (i % 2)));
        return f16 ? (float)f16_from_bits(b) : bf16_to_f32(b);
    }
};

// Keys of pages [page0, page1) of a row, by the workgroup's threads: `put(page, key)`.
template <bool WIDE, typename PUT>
EP_DEV void score_pages(const SelectArgs &a, const SelectRow &row, int64_t page0, int64_t page1, PUT put)
{
    const int L = a.lanes, tid = threadIdx.x, u = tid & (L - 1), D = a.c.D;
    const bool in = 8 * u < D;
    const int d = in ? 8 * u : 0;
    const int32_t *table = a.tok.table + row.b * a.tok.table_stride;
    const int step = (int)blockDim.x / L;
    int64_t k0 = page0 + tid / L;
    int32_t id[2];
    auto load_ids = [&]() {
#pragma unroll
        for (int k = 0; k < 2; ++k)      // past the end some page of the row's
            id[k] = table[k0 + k * step < page1 ? k0 + k * step : page0];
    };
    load_ids();
    // this lane's eight columns of the group's queries, four heads in flight
    double up[8], down[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        up[i] = down[i] = 0.0;
    const char *q = (const char *)a.q + 2 * (row.b * a.q_sb + row.s * a.q_ss + (int64_t)row.h * a.G * a.q_sh + d);
    for (int g0 = 0; g0 < a.G; g0 += 4) {
        u32x4_t w[4];
#pragma unroll
        for (int g = 0; g < 4; ++g)
            w[g] = *(const u32x4_t *)(q + 2 * (g0 + g < a.G ? g0 + g : g0) * a.q_sh);
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (g0 + g < a.G)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint16_t x = (uint16_t)(w[g][i / 2] >> (16 * (i % 2)));
                    const float v = a.q_dtype == EP_F16 ? (float)f16_from_bits(x) : bf16_to_f32(x);
                    // a NaN reaches both sums
                    up[i] += v < 0.0f ? 0.0 : (double)v;
                    down[i] += v > 0.0f ? 0.0 : (double)v;
                }
    }
    const bool f16 = a.c.dtype == EP_F16;
    while (k0 < page1) {
        Bounds8<WIDE> lo[2], hi[2];
        bool ok[2];
        const int64_t at = k0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            ok[k] = id[k] >= 0 && id[k] < a.c.n_pages;
            const int64_t src = ((int64_t)(ok[k] ? id[k] : 0) * a.c.heads + row.h) * 2 * D + d;
            lo[k].load(a.bounds, src);
            hi[k].load(a.bounds, src + D);
        }
        k0 += 2 * step;
        load_ids();      // of the next round, while this one's bounds are on their way
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                sum = fma((double)lo[k].at(i, f16), down[i], fma((double)hi[k].at(i, f16), up[i], sum));
            sum = lanes_sum(in ? sum : 0.0, L);
            if (u == 0 && at + k * step < page1)
                put(at + k * step, ok[k] ? order_key(sum) : ~0ull);
        }
    }
}

template <bool WIDE>
__global__ void __launch_bounds__(256) score_kernel(SelectArgs a)
{
    const uint32_t at = a.first_wg + blockIdx.x, r = at / a.chunks, chunk = at - r * a.chunks;
    const SelectRow row = select_row(a, r);
    const int64_t page0 = (int64_t)chunk * kChunkPages, page1 = page0 + kChunkPages < row.own ? page0 + kChunkPages : row.own;
    if (row.own < a.take || page0 >= page1)      // all pages are taken, or none of these is asked about
        return;
    uint64_t *keys = a.keys + (int64_t)r * a.tok.width;
    score_pages<WIDE>(a, row, page0, page1, [&](int64_t page, uint64_t key) { keys[page] = key; });
}

constexpr int kChoose = 512;        // threads of a row's choice
constexpr int kChooseWaves = kChoose / 64, kDigits = 2048;

// Exclusive sums over the workgroup's threads of two counts.
EP_DEV uint2 exclusive_sums(uint32_t x, uint32_t y, uint2 *s_part)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t px = x, py = y;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t ox = __shfl_up(px, d, 64), oy = __shfl_up(py, d, 64);
        px += lane >= d ? ox : 0u;
        py += lane >= d ? oy : 0u;
    }
    __syncthreads();
    if (lane == 63)
        s_part[wave] = make_uint2(px, py);
    __syncthreads();
    uint2 before = make_uint2(px - x, py - y);
#pragma unroll
    for (int w = 0; w < kChooseWaves; ++w) {
        before.x += w < wave ? s_part[w].x : 0u;
        before.y += w < wave ? s_part[w].y : 0u;
    }
    return before;
}

struct ChooseShared {
    uint32_t count[kDigits];
    uint64_t least[kChooseWaves], largest[kChooseWaves];
    uint2 part[kChooseWaves];
    uint32_t found[3];
};

// The (take - 1) largest of n keys, in order, and page n behind them: found
// digit by digit from the top.  A round counts 2048 digits of what lies
// between the least and the largest key still in question, so that the first
// one parts them about as well as their number allows; of equal keys the first
// are taken.  lo, hi: the least and the largest of the keys that this thread
// has seen.
template <typename KEY>
EP_DEV void choose(ChooseShared &sh, int64_t n, int take, uint64_t lo, uint64_t hi, KEY key, int32_t *out)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) {
        const uint64_t l = __shfl_xor(lo, d, 64), h = __shfl_xor(hi, d, 64);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
    }
    if (lane == 0) {
        sh.least[wave] = lo;
        sh.largest[wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kChooseWaves; ++w) {
        lo = sh.least[w] < lo ? sh.least[w] : lo;
        hi = sh.largest[w] > hi ? sh.largest[w] : hi;
    }
    uint64_t span = hi - lo;
    uint32_t need = take - 1;
    bool all = false;        // every key from lo on is taken; else `need` of those equal to lo
    for (;;) {
        const int bits = span ? 64 - __builtin_clzll(span) : 0, shift = bits > 11 ? bits - 11 : 0;
        for (int i = tid; i < kDigits; i += kChoose)
            sh.count[i] = 0;
        __syncthreads();
        for (int64_t i = tid; i < n; i += kChoose) {
            const uint64_t k = key(i) - lo;         // below lo: past the span
            if (k <= span)
                atomicAdd(&sh.count[k >> shift], 1u);
        }
        __syncthreads();
        // thread t holds the digits from kDigits - 1 - E t down
        constexpr int E = kDigits / kChoose;
        uint32_t c[E], sum = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            c[i] = sh.count[kDigits - 1 - E * tid - i];
            sum += c[i];
        }
        uint32_t above = exclusive_sums(sum, 0, sh.part).x;
        if (above < need && above + sum >= need)
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if (above < need && above + c[i] >= need) {
                    sh.found[0] = kDigits - 1 - E * tid - i;
                    sh.found[1] = above;
                    sh.found[2] = c[i];
                }
                above += c[i];
            }
        __syncthreads();
        lo += (uint64_t)sh.found[0] << shift;
        need -= sh.found[1];
        all = sh.found[2] == need;
        if (all || shift == 0)
            break;
        span = (1ull << shift) - 1;
    }
    // in order: thread t writes what it takes of its n / kChoose keys
    const int64_t per = (n + kChoose - 1) / kChoose, i0 = tid * per < n ? tid * per : n, i1 = i0 + per < n ? i0 + per : n;
    uint32_t over = 0, equal = 0;
    for (int64_t i = i0; i < i1; ++i) {
        const uint64_t k = key(i);
        over += all ? k >= lo : k > lo;
        equal += !all && k == lo;
    }
    const uint2 before = exclusive_sums(over, equal, sh.part);
    uint32_t ties = before.y, to = before.x + (all ? 0u : ties < need ? ties : need);
    for (int64_t i = i0; i < i1; ++i) {
        const uint64_t k = key(i);
        bool in = all ? k >= lo : k > lo;
        if (!all && k == lo)
            in = ties++ < need;
        if (in)
            out[to++] = (int32_t)i;
    }
    if (tid == 0)
        out[take - 1] = (int32_t)n;
}

// A row whose pages are all taken, or of which only its own is: done, true.
EP_DEV bool chosen_at_once(int64_t n, int take, int32_t *out)
{
    if (n >= take && take > 1)
        return false;
    for (int i = threadIdx.x; i < take; i += kChoose)
        out[i] = n >= take ? (int32_t)n : i <= n ? i : -1;
    return true;
}

// A row's choice among scores in memory.
__global__ void __launch_bounds__(kChoose) choose_kernel(SelectArgs a)
{
    __shared__ uint64_t s_key[kHeldKeys];
    __shared__ ChooseShared sh;
    const uint32_t r = a.first_wg + blockIdx.x;
    const int64_t n = select_row(a, r).own;
    int32_t *out = a.blocks + (int64_t)r * a.take;
    if (chosen_at_once(n, a.take, out))
        return;
    const uint64_t *keys = a.keys + (int64_t)r * a.tok.width;
    const bool held = n <= kHeldKeys;
    uint64_t lo = ~0ull, hi = 0;
    for (int64_t i0 = threadIdx.x; i0 < n; i0 += 4 * kChoose) {
        uint64_t k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)      // four loads in flight; past the end the first again
            k[i] = keys[i0 + i * kChoose < n ? i0 + i * kChoose : i0];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (held && i0 + i * kChoose < n)
                s_key[i0 + i * kChoose] = k[i];
            lo = k[i] < lo ? k[i] : lo;
            hi = k[i] > hi ? k[i] : hi;
        }
    }
    choose(sh, n, a.take, lo, hi, [&](int64_t i) { return held ? s_key[i] : keys[i]; }, out);
}

// Scores and choice of a row in one workgroup, where its pages are few.
template <bool WIDE>
__global__ void __launch_bounds__(kChoose) select_kernel(SelectArgs a)
{
    __shared__ uint64_t s_key[kFewPages];
    __shared__ ChooseShared sh;
    const uint32_t r = a.first_wg + blockIdx.x;
    const SelectRow row = select_row(a, r);
    int32_t *out = a.blocks + (int64_t)r * a.take;
    if (chosen_at_once(row.own, a.take, out))
        return;
    uint64_t lo = ~0ull, hi = 0;
    score_pages<WIDE>(a, row, 0, row.own, [&](int64_t page, uint64_t key) {
        s_key[page] = key;
        lo = key < lo ? key : lo;
        hi = key > hi ? key : hi;
    });
    choose(sh, row.own, a.take, lo, hi, [&](int64_t i) { return s_key[i]; }, out);
}

// A launch has fewer than 2^32 threads: a grid beyond that is cut into several.
template <typename ARGS, typename F>
int in_launches(int64_t grid, unsigned threads, ARGS a, F launch)
{
    const int64_t most = 0xffffffff / threads;
    for (int64_t at = 0; at < grid; at += most) {
        a.first_wg = (uint32_t)at;
        launch(a, (unsigned)(grid - at < most ? grid - at : most));
        EP_HIP_CHECK(hipGetLastError());
    }
    return EP_OK;
}

}  // namespace

int launch_kv_bounds(const PagedTokens &tok, const PagedCache &c, void *bounds, int64_t limit, hipStream_t stream)
{
    // From 1024 pages and heads on a wave rebuilds a page alone.  With four / one,
    // 8 heads of 128 in bf16, append included: 2 x 512 tokens on pages of 64, 128 of
    // them, 12.1 / 15.4 us; 2 x 2048, 512, 19.1 / 21.7; 3 x 2048, 768, 23.0 / 24.0;
    // 2 x 4096, 1024, 28.5 / 26.2; on pages of 16 2 x 512, 512, 23.0 / 21.9; 2 x 4096,
    // 4096, 43 / 33; 65536, 32768, 349 / 173.
    const bool alone = tok.S > 1 && tok.B * c.heads * ((tok.S + c.page - 1) >> c.page_shift) >= 1024;
    // Every workgroup looks at its whole row for the positions' order: long rows
    // have no more than kRowChunks of them a head.
    const int64_t tokens = (tok.S + kGroupTokens - 1) / kGroupTokens;
    const int64_t each = std::max<int64_t>((tokens + kRowChunks - 1) / kRowChunks, alone ? 4 : 1);
    const int64_t chunks = (tokens + each - 1) / each;
    const int64_t parts = tok.B * chunks;
    if (parts > 0x7fffffff / c.heads)
        return set_error(EP_DECLINE_SHAPE, "bounds of %lld x %lld tokens are more than one call takes", (long long)tok.B,
                         (long long)tok.S);
    // What a workgroup finds out about its tokens holds for all heads, and a look at
    // the other sequences grows with their number: more workgroups than 4096 take
    // several heads each.  One head / so, 8 heads of 128 in bf16, append included:
    // 512 x 1 tokens 19.7 / 20.6 us (the kernel's registers), 2048 x 1 68 / 60,
    // 4096 x 1 162 / 113, 4096 x 4 358 / 128.
    const int64_t some = std::max<int64_t>(1, std::min<int64_t>(c.heads, parts * c.heads / 4096));
    const int64_t head_groups = (c.heads + some - 1) / some;
    const BoundsArgs args{tok, c, bounds, limit, 0, (uint32_t)chunks, (uint32_t)each, (uint32_t)some, (uint32_t)head_groups};
    auto run = [&](auto code) {
        constexpr int CODE = decltype(code)::value;
        return in_launches(parts * head_groups, 256, args, [&](const BoundsArgs &a, unsigned n) {
            if (tok.S == 1)
                bounds_kernel<CODE, 0><<<n, 256, 0, stream>>>(a);
            else if (alone)
                bounds_kernel<CODE, 1><<<n, 256, 0, stream>>>(a);
            else
                bounds_kernel<CODE, 4><<<n, 256, 0, stream>>>(a);
        });
    };
    switch (c.dtype) {
    case EP_BF16: return run(std::integral_constant<int, EP_BF16>());
    case EP_F16: return run(std::integral_constant<int, EP_F16>());
    case EP_I8: return run(std::integral_constant<int, EP_I8>());
    default: return run(std::integral_constant<int, EP_E4M3>());
    }
}

// No scores in memory where every page is taken, or pages are few.
size_t select_workspace(const PagedTokens &tok, const PagedCache &c, int64_t take)
{
    return tok.width > take && take > 1 && tok.width > kFewPages ? (size_t)tok.B * tok.S * c.heads * tok.width * sizeof(uint64_t) : 0;
}

int launch_kv_select(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, const void *bounds, int64_t take,
                     int32_t *blocks, void *ws, size_t ws_bytes, hipStream_t stream)
{
    const int64_t rows = tok.B * tok.S * c.heads, chunks = (tok.width + kChunkPages - 1) / kChunkPages;
    if (rows > 0x7fffffff || (chunks > 0 && rows > 0x7fffffff / chunks))
        return set_error(EP_DECLINE_SHAPE, "%lld rows over %lld pages are more than one call takes", (long long)rows,
                         (long long)tok.width);
    const size_t want = select_workspace(tok, c, take);
    if (ws_bytes < want || (want && !ws))
        return set_error(EP_ERR_WORKSPACE, "select: workspace of %zu bytes, %zu wanted", ws_bytes, want);
    SelectArgs a{};
    a.q = q->ptr;
    a.q_sb = q->stride_b;
    a.q_ss = q->stride_s;
    a.q_sh = q->stride_h;
    a.q_dtype = q->dtype;
    a.G = q->heads / c.heads;
    a.tok = tok;
    a.c = c;
    a.bounds = bounds;
    a.keys = (uint64_t *)ws;
    a.blocks = blocks;
    a.chunks = (uint32_t)chunks;
    a.take = (int)take;
    a.lanes = 2;
    while (a.lanes * 8 < c.D)
        a.lanes *= 2;
    const bool wide = c.dtype != EP_F16 && c.dtype != EP_BF16;
    if (!want)
        return in_launches(rows, kChoose, a, [&](const SelectArgs &part, unsigned n) {
            if (wide)
                select_kernel<true><<<n, kChoose, 0, stream>>>(part);
            else
                select_kernel<false><<<n, kChoose, 0, stream>>>(part);
        });
    int rc = in_launches(rows * chunks, 256, a, [&](const SelectArgs &part, unsigned n) {
        if (wide)
            score_kernel<true><<<n, 256, 0, stream>>>(part);
        else
            score_kernel<false><<<n, 256, 0, stream>>>(part);
    });
    if (rc == EP_OK)
        rc = in_launches(rows, kChoose, a, [&](const SelectArgs &part, unsigned n) { choose_kernel<<<n, kChoose, 0, stream>>>(part); });
    return rc;
}

}  // namespace ep
