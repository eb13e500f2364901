// Attention of a whole batch's rows over the pages that its tables begin with
// (attend.hip plans and joins; attend_gen_front.hip instantiates).
//
// Many rows meet every key here, so a tile of keys and values is brought to LDS
// once a workgroup and read from there by all of its waves: 128 rows (token by
// token, the group's query heads side by side), a stage of 64 or 128
// positions, four waves of 32 rows each, or eight of which two share the rows
// and halve the stage.  The next stage's rows are in flight while this one is
// multiplied.
//
// The products are those of attend_kernel.h: S^T = K Q^T gives lane (n, g) the
// scores of positions 16 t + 4 g + i of query row n, which is the operand of
// O^T = V^T P^T if its index 8 g + 4 t + i means position 16 t + 4 g + i: what a
// transposing LDS read of four rows gives.  16-bit rows go to LDS past the
// registers; codes of 8 bits become 16-bit values on the way, once for all
// rows.  Rounding as there.
#pragma once

#include "attend_kernel.h"

namespace ep {

constexpr int kFrontRows = 128;

struct FrontArgs {
    const void *q;
    int64_t q_sb, q_ss, q_sh;
    PagedTokens tok;
    PagedCache c;
    float scale;             // of the scores, times log2(e)
    int window, cap;
    int G, rows;             // query heads a cache head; rows of the batch on one of them
    int limit;               // positions on the shared pages
    int groups, splits;      // of kFrontRows rows; pieces of the positions
    uint32_t first_wg;
    float2 *part_ml;         // [groups][heads][splits][kFrontRows]: maximum, sum
    float *part_o;           // [groups][heads][splits][kFrontRows][D]
};

// Positions of a stage: two of them fill LDS.  Waves: two a SIMD as long as
// their sums fit half of the registers.
// 8-bit rows pass through registers, so fewer of them are in flight.
constexpr int front_stage(int KS, bool k8) { return KS <= 3 ? 128 : k8 ? (KS == 8 ? 32 : 64) : KS == 4 ? 128 : 64; }
constexpr int front_waves(int KS) { return KS <= 4 ? 8 : 4; }

// Where chunk c (eight values, 16 bytes) of row r of a stage lies in its row of
// 4 KS chunks: the rows of one read (16 adjacent ones, at the same columns) lie
// on different banks.
template <int KS>
EP_DEV int front_chunk(int r, int c)
{
    return c ^ (KS % 4 == 0 ? r & 15 : KS == 3 ? (r >> 2) & 3 : (r >> 1) & 7);
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));

// Read by lanes for what is not there.
__device__ const u32x4_t kFrontZeros = {0, 0, 0, 0};

template <typename QOP, int CODE, int KS>
__global__ void __launch_bounds__(64 * front_waves(KS), front_waves(KS) / 4) front_kernel(FrontArgs a)
{
    constexpr bool k8 = CODE == EP_I8 || CODE == EP_E4M3;
    constexpr int ES = k8 ? 1 : 2, NC = 2 * KS, DM = 32 * KS, TP = front_stage(KS, k8);
    constexpr int WAVES = front_waves(KS), THREADS = 64 * WAVES, HALVES = WAVES / 4, IDS = TP / 16;
    constexpr int NK = TP * 4 * KS / THREADS;        // a thread's chunks of a stage's keys, and of its values
    static_assert(NK * THREADS == TP * 4 * KS, "whole chunks");
    using VOP = typename std::conditional<k8, OpBf16, QOP>::type;
    // A stage's keys, then its values; scales.  The two stages are arrays of
    // their own: the compiler waits for rows on their way into an array before
    // it reads from it.
    __shared__ __attribute__((aligned(16))) uint16_t s_even[2 * TP * DM], s_odd[2 * TP * DM];
    __shared__ float s_ks[2][k8 ? TP : 1], s_vs[2][k8 ? TP : 1];
    __shared__ float2 s_ml[HALVES == 1 ? 1 : 4][16];
    __shared__ int s_id[4][IDS], s_lo[4], s_hi[4];      // page ids of four stages, 16 positions each

    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave / HALVES, half = wave % HALVES;
    const int H = a.c.heads, D = a.c.D;
    const float nan = __uint_as_float(0x7fc00000u);
    // Workgroups go to the eight XCDs in turn: those that read one piece of one
    // head (its row groups) share an XCD's L2.
    const uint32_t pairs = (uint32_t)H * a.splits;
    uint32_t pair, group;
    {
        const uint32_t wg = a.first_wg + blockIdx.x, x = wg & 7, y = wg >> 3;
        pair = (y / a.groups) * 8 + x;
        group = y % a.groups;
    }
    if (pair >= pairs)
        return;
    const int h = pair % (uint32_t)H, split = pair / (uint32_t)H;
    const int row0 = group * kFrontRows + 32 * rw, row_end = a.rows;

    // ---- rows: what they see, their queries
    int first[2], last[2], pos[2];
    int64_t q_at[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        const int row = min(row0 + 16 * mt + n, row_end - 1);
        const int t = (uint32_t)row / (uint32_t)a.G, head = row - t * a.G;
        const uint32_t b = (uint32_t)t / (uint32_t)a.tok.S, s = t - b * (uint32_t)a.tok.S;
        const int64_t p = a.tok.pos[b * a.tok.pos_sb + s * a.tok.pos_ss];
        pos[mt] = row0 + 16 * mt + n >= row_end || p < 0 || p >= a.cap ? -1 : (int)p;
        q_at[mt] = b * a.q_sb + s * a.q_ss + (int64_t)(h * a.G + head) * a.q_sh;
    }
    u32x4_t q[2][KS];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d = 32 * k + 8 * g;
            q[mt][k] = *(const u32x4_t *)((const char *)a.q + 2 * (q_at[mt] + (d < D ? d : 0)));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                q[mt][k][i] = d < D ? q[mt][k][i] : 0u;
        }
    int lo = -a.cap, hi = -1, in_lo = 0, in_hi = -a.cap;         // over the wave's rows: seen by any (lo negated), by all
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        const int p = pos[mt];
        first[mt] = p >= a.window ? p - a.window + 1 : 0;
        last[mt] = min(p, a.limit - 1);
        const bool some = p >= 0 && first[mt] <= last[mt];
        first[mt] = some ? first[mt] : a.cap;
        last[mt] = some ? last[mt] : -1;
        lo = max(lo, some ? -first[mt] : -a.cap);
        hi = max(hi, last[mt]);
        in_lo = max(in_lo, some ? first[mt] : p >= 0 ? a.cap : 0);       // a row that sees nothing masks every tile
        in_hi = max(in_hi, some ? -last[mt] : -a.cap);
    }
    lo = -dpp_row_max(lo);
    hi = dpp_row_max(hi);
    in_lo = dpp_row_max(in_lo);
    in_hi = -dpp_row_max(in_hi);
    const bool ragged = lo != in_lo || hi != in_hi;
    if (lane == 0 && half == 0) {
        s_lo[rw] = lo;
        s_hi[rw] = hi;
    }
    __syncthreads();
    const int all_lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3])), all_hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
    // stages that the group's rows reach, this piece's share of them
    int j = 0, end = 0;
    if (all_hi >= 0) {
        const int j0 = all_lo / TP, stages = all_hi / TP + 1 - j0;
        j = j0 + (int)((int64_t)stages * split / a.splits);
        end = j0 + (int)((int64_t)stages * (split + 1) / a.splits);
    }

    // ---- staging: chunk x of the stage in LDS (x = row, place in it) is a thread's x % THREADS == tid
    uint2 kr[k8 ? NK : 1], vr[k8 ? NK : 1];
    float sr[2];
    auto page_of = [&](int p) { return a.tok.table[min(p, a.limit - 1) >> a.c.page_shift]; };
    // Row in the pool of position `at` of stage j; -1: none
    auto row_of = [&](int j, int at) -> int64_t {
        const int id = s_id[j & 3][at / 16], p = j * TP + at;
        const int64_t row = ((int64_t)id * H + h) * a.c.page + (p & (a.c.page - 1));
        return (int)(p < a.limit) & (int)(id >= 0) & (int)(id < a.c.n_pages) ? row : -1;      // no branch
    };
    auto stage = [&](auto odd) -> uint16_t * {
        if constexpr (decltype(odd)::value)
            return s_odd;
        else
            return s_even;
    };
    auto load_rows = [&](auto odd, int j) {
        uint16_t *const dst = stage(odd);
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int x = tid + THREADS * i, r = x / (4 * KS), c = front_chunk<KS>(r, x % (4 * KS));
            const int64_t row = row_of(j, r);
            const bool ok = (int)(row >= 0) & (int)(8 * c < D);
            const int64_t at = (row * D + 8 * c) * ES;
            const char *ks = ok ? (const char *)a.c.k + at : (const char *)&kFrontZeros;
            const char *vs = ok ? (const char *)a.c.v + at : (const char *)&kFrontZeros;
            if constexpr (k8) {
                kr[i] = *(const uint2 *)ks;
                vr[i] = *(const uint2 *)vs;
            } else {
                const int x0 = 8 * (64 * wave + THREADS * i);        // lane l writes 16 bytes at 16 l from there
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)ks,
                                                 (__attribute__((address_space(3))) void *)&dst[x0], 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)vs,
                                                 (__attribute__((address_space(3))) void *)&dst[TP * DM + x0], 16, 0, 0);
            }
        }
        if constexpr (k8)
            if (tid < TP) {
                const int64_t row = row_of(j, tid);
                sr[0] = a.c.k_scale[row >= 0 ? row : 0];
                sr[1] = a.c.v_scale[row >= 0 ? row : 0];
                sr[0] = row >= 0 ? sr[0] : 0.0f;
                sr[1] = row >= 0 ? sr[1] : 0.0f;
            }
    };
    auto store_rows = [&](auto odd) {
        if constexpr (k8) {
            uint16_t *const dst = stage(odd);
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const int x = tid + THREADS * i;
                *(u32x4_t *)&dst[8 * x] = decode8<QOP, CODE>(kr[i].x, kr[i].y);
                *(u32x4_t *)&dst[TP * DM + 8 * x] = decode8<VOP, CODE>(vr[i].x, vr[i].y);
            }
            if (tid < TP) {
                s_ks[decltype(odd)::value][tid] = sr[0];
                s_vs[decltype(odd)::value][tid] = sr[1];
            }
        }
    };

    // ---- the running softmax
    float m[2], l[2];
    f32x4_t o[2][NC];
    // Outputs that a value which is not finite has reached: written into the
    // sums where it happens, or, in wide heads, a bit each (the sums' registers
    // do not fit twice: 76 of 256 values would go through memory).
    constexpr bool kHitsApart = KS > 4;
    uint32_t hit[2][(NC + 7) / 8] = {};
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        m[mt] = -INFINITY;
        l[mt] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            o[mt][c] = (f32x4_t){0, 0, 0, 0};
    }
    // 32 positions from j0, `at` in the stage.  edge: some row sees them in part, or
    // a page is missing, so that scores are masked one by one.
    auto tile = [&](auto odd, auto edge_type, int at, int j0, bool bad0, bool bad1) {
        constexpr bool edge = decltype(edge_type)::value;
        constexpr int buf = decltype(odd)::value;
        const uint16_t *const keys = stage(odd);
        uint16_t *const values = stage(odd) + TP * DM;
        f32x4_t sc[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            sc[0][t] = sc[1][t] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const int r = at + 16 * t + n;
                const u32x4_t f = *(const u32x4_t *)&keys[r * DM + 8 * front_chunk<KS>(r, 4 * k + g)];
                sc[0][t] = QOP::mfma(f, q[0][k], sc[0][t]);
                sc[1][t] = QOP::mfma(f, q[1][k], sc[1][t]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);       // each phase's LDS reads stay in it: their registers are not there twice
        float vs[8];
        float x[2][8];
        if constexpr (k8) {
            float ks[8];
            __builtin_memcpy(ks, __builtin_assume_aligned(&s_ks[buf][at + 4 * g], 16), 16);
            __builtin_memcpy(ks + 4, __builtin_assume_aligned(&s_ks[buf][at + 16 + 4 * g], 16), 16);
            __builtin_memcpy(vs, __builtin_assume_aligned(&s_vs[buf][at + 4 * g], 16), 16);
            __builtin_memcpy(vs + 4, __builtin_assume_aligned(&s_vs[buf][at + 16 + 4 * g], 16), 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ks[e] *= a.scale;
                x[0][e] = sc[0][e / 4][e % 4] * ks[e];
                x[1][e] = sc[1][e / 4][e % 4] * ks[e];
            }
        } else
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[mt][e] = sc[mt][e / 4][e % 4] * a.scale;
        uint32_t seen[2] = {0xff, 0xff};
        if constexpr (edge)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                seen[mt] = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int p = j0 + 16 * (e / 4) + 4 * g + e % 4;
                    const bool in = p >= first[mt] && p <= last[mt];
                    seen[mt] |= (uint32_t)in << e;
                    x[mt][e] = !in ? -INFINITY : (e < 4 ? bad0 : bad1) ? nan : x[mt][e];
                }
            }
        u32x4_t ph[2], pl[2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            float top = x[mt][0];
#pragma unroll
            for (int e = 1; e < 8; ++e)
                top = fmaxf(top, x[mt][e]);
            top = fmaxf(m[mt], xor32_max(xor16_max(top)));
            const float base = top == -INFINITY ? 0.0f : top;
            if (__any(top > m[mt])) {
                const float keep = __builtin_amdgcn_exp2f(m[mt] - base);
                l[mt] *= keep;
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[mt][c][i] *= keep;
            }
            m[mt] = top;
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = x[mt][e] - base;
                if constexpr (VOP::kShift != 0.0f)
                    w[e] += VOP::kShift;         // on the difference: a score past 2^24 would round it away
                w[e] = __builtin_amdgcn_exp2f(w[e]);
                l[mt] += w[e];
                if constexpr (k8)
                    w[e] = edge && !(seen[mt] >> e & 1) ? 0.0f : w[e] * vs[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ph[mt][e] = VOP::pack(w[2 * e], w[2 * e + 1]);
                pl[mt][e] = VOP::pack(w[2 * e] - VOP::low(ph[mt][e]), w[2 * e + 1] - VOP::high(ph[mt][e]));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        // Values that no row sees become zero; what some rows see and others not
        // is taken out if it is not finite, and added where it is seen.
        u32x4_t keep, one[2];
        if constexpr (edge)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = j0 + 16 * (e / 2) + 4 * g + 2 * (e % 2);
                keep[e] = (p >= lo && p <= hi ? 0xffffu : 0u) | (p + 1 >= lo && p + 1 <= hi ? 0xffff0000u : 0u);
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
                    one[mt][e] = (seen[mt] >> (2 * e) & 1 ? VOP::kOne : 0u) | (seen[mt] >> (2 * e + 1) & 1 ? VOP::kOne << 16 : 0u);
            }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c % 4 == 0 && c > 0)
                __builtin_amdgcn_sched_barrier(0);
            // column 16 c + n of rows 4 g + i, and of those 16 behind: a lane names a quarter of row n / 4 of its four
            u32x4_t f;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int r = at + 16 * t + 4 * g + n / 4;
                const s16x4_t w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4_t *)&values[r * DM + 8 * front_chunk<KS>(r, 2 * c + (n >> 1 & 1)) + 4 * (n & 1)]);
                uint2 u;
                __builtin_memcpy(&u, &w, 8);
                f[2 * t] = u.x;
                f[2 * t + 1] = u.y;
            }
            if constexpr (edge) {
                u32x4_t odd;
                uint32_t some = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[e] &= keep[e];
                    odd[e] = CODE == EP_I8 || !ragged ? 0u : not_finite<VOP::kDtype>(f[e]);
                    some |= odd[e];
                    f[e] &= ~odd[e];
                    odd[e] &= VOP::kOne | VOP::kOne << 16;
                }
                if (CODE != EP_I8 && __any(some != 0))
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        const f32x4_t hits = VOP::mfma(odd, one[mt], (f32x4_t){0, 0, 0, 0});
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if constexpr (kHitsApart)
                                hit[mt][c / 8] |= (hits[i] > 0.0f ? 1u : 0u) << (4 * (c % 8) + i);
                            else
                                o[mt][c][i] = hits[i] > 0.0f ? nan : o[mt][c][i];
                    }
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
                o[mt][c] = VOP::mfma(f, pl[mt], VOP::mfma(f, ph[mt], o[mt][c]));
        }
    };

    // The stage's tiles of one kind.
    auto tiles = [&](auto odd, auto edge) {
#pragma unroll 1
        for (int i = 0; i < TP / 32 / HALVES; ++i) {
            const int at = (TP / HALVES) * half + 32 * i, j0 = j * TP + at;
            const int id0 = __builtin_amdgcn_readfirstlane(s_id[j & 3][at / 16]);
            const int id1 = __builtin_amdgcn_readfirstlane(s_id[j & 3][at / 16 + 1]);
            const bool bad0 = id0 < 0 || id0 >= a.c.n_pages, bad1 = id1 < 0 || id1 >= a.c.n_pages;
            const bool some = j0 <= hi && j0 + kAttTile > lo, cut = j0 < in_lo || j0 + kAttTile - 1 > in_hi || bad0 || bad1;
            if (some && cut == decltype(edge)::value)
                tile(odd, edge, at, j0, bad0, bad1);
        }
    };
    // Stage j, the next one on its way meanwhile.
    auto step = [&](auto odd, auto next) {
        const bool more = j + 1 < end;
        int id = 0;
        if (more) {
            load_rows(next, j + 1);
            if (tid < IDS)
                id = page_of((j + 2) * TP + 16 * tid);
        }
        tiles(odd, std::false_type());
        tiles(odd, std::true_type());
        if (more) {
            store_rows(next);
            if (tid < IDS)
                s_id[(j + 2) & 3][tid] = id;
        }
        __syncthreads();         // the next stage is there, and this one's readers are done
        ++j;
    };
    if (j < end) {
        if (tid < 2 * IDS)
            s_id[(j + tid / IDS) & 3][tid % IDS] = page_of(j * TP + 16 * tid);
        __syncthreads();
        load_rows(std::false_type(), j);
        store_rows(std::false_type());
        __syncthreads();
        for (;;) {
            step(std::false_type(), std::true_type());
            if (j >= end)
                break;
            step(std::true_type(), std::false_type());
            if (j >= end)
                break;
        }
    }

    // ---- the two halves' parts joined, and left
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        l[mt] = xor32_sum(xor16_sum(l[mt]));
        if constexpr (kHitsApart)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[mt][c][i] = hit[mt][c / 8] >> (4 * (c % 8) + i) & 1 ? nan : o[mt][c][i];
    }
    const int64_t slot = ((int64_t)group * H + h) * a.splits + split;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        float2 other = make_float2(-INFINITY, 0.0f);
        f32x4_t *so = (f32x4_t *)s_even + rw * NC * 64;      // waves of the second half hand over there
        if constexpr (HALVES > 1) {
            static_assert(4 * NC * 64 * 16 <= (int)sizeof s_even, "a stage holds the hand-over");
            if (half) {
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    so[c * 64 + lane] = o[mt][c];
                if (g == 0)
                    s_ml[rw][n] = make_float2(m[mt], l[mt]);
            }
            __syncthreads();
            other = s_ml[rw][n];
        }
        const int r = 32 * rw + 16 * mt + n;
        if (!half && group * kFrontRows + r < row_end) {
            const float top = fmaxf(m[mt], other.x), base = top == -INFINITY ? 0.0f : top;
            const float f0 = __builtin_amdgcn_exp2f(m[mt] - base), f1 = __builtin_amdgcn_exp2f(other.x - base);
            const int64_t at = slot * kFrontRows + r;
            if (g == 0)
                a.part_ml[at] = make_float2(top, l[mt] * f0 + other.y * f1);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                f32x4_t z = o[mt][c];
                if constexpr (HALVES > 1) {
                    const f32x4_t y = so[c * 64 + lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        z[i] = z[i] * f0 + y[i] * f1;
                }
                if (16 * c < D)
                    *(f32x4_t *)(a.part_o + at * D + 16 * c + 4 * g) = z;
            }
        }
        if constexpr (HALVES > 1)
            __syncthreads();
    }
}

// Steps of 32 values that a kernel takes for heads of D values.
constexpr int front_steps(int D) { return D <= 64 ? 2 : D <= 96 ? 3 : D <= 128 ? 4 : D <= 192 ? 6 : 8; }

template <typename QOP, int CODE, int KS>
void front_sized(const FrontArgs &a, unsigned grid, hipStream_t st)
{
    front_kernel<QOP, CODE, KS><<<grid, 64 * front_waves(KS), 0, st>>>(a);
}
template <typename QOP, int CODE>
void front_by_size(const FrontArgs &a, unsigned grid, hipStream_t st)
{
    switch (front_steps(a.c.D)) {
    case 2: return front_sized<QOP, CODE, 2>(a, grid, st);
    case 3: return front_sized<QOP, CODE, 3>(a, grid, st);
    case 4: return front_sized<QOP, CODE, 4>(a, grid, st);
    case 6: return front_sized<QOP, CODE, 6>(a, grid, st);
    default: return front_sized<QOP, CODE, 8>(a, grid, st);
    }
}

void attend_front(const FrontArgs &a, int q_dtype, unsigned grid, hipStream_t st);

}  // namespace ep
