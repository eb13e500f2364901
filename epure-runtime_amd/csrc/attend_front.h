// Attention of a whole batch's rows over the pages that its tables begin with
// (attend.hip plans and joins; attend_gen_front.hip and attend_gen_tails.hip instantiate).
//
// Many rows meet every key here, so a stage of 64 positions' keys and values is
// brought to LDS once a workgroup and read from there by all of its four waves:
// 128 rows (token by token, the group's query heads side by side), 32 a wave.
// Two stages lie in LDS, one on its way while the other is read; a compute unit
// holds two workgroups, so that one has something to do where the other waits.
//
// The products are those of attend_kernel.h: S^T = K Q^T gives lane (n, g) the
// scores of positions 16 t + 4 g + i of query row n, which is the operand of
// O^T = V^T P^T if its index 8 g + 4 t + i means position 16 t + 4 g + i: what a
// transposing LDS read of four rows gives.  16-bit rows go from memory to LDS
// past the registers; codes of 8 bits become 16-bit values on the way, once for
// all rows.  Rounding as there: the weights' second term costs more here (28 of
// the 120 us below), and is kept so that a token's answer does not lose bits with
// the company that it is computed in.
//
// Bound by vector and matrix instructions that hardly overlap.  64 sequences of 4
// query heads on each of 8 cache heads over 65536 positions of 128 (bf16: 268 MB,
// 103 GFLOP of products with the second term): 120 us, 106 with nothing loaded.  The
// instructions counted, at the clocks of each kind in a loop of its own, are some 70
// us of vector ones and 60 of matrix ones: about their sum is what is measured.  One
// workgroup of eight waves a compute unit and stages of 128 positions took 182.  128
// such sequences over 16384 positions in int8: 75.  Wider heads are not taken: two
// workgroups' stages of 64 positions, and 32 rows a wave, leave them no room.
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

constexpr int kFrontWaves = 4, kFrontStage = 64;

// Workgroups that a compute unit holds, and the widest heads.  Those of 128 values
// take all registers that two leave them: nine of the kernels put two or three more
// away (12 bytes of scratch a lane).
constexpr int kFrontOccupancy = 2, kFrontWidest = 128;

// How far (in powers of two) a row's weights may outgrow the maximum that they
// are taken relative to before sums and maximum are brought up to date: most
// stages then leave them alone.  f16 weights stay below 2^15 with it.
constexpr float front_slack(float shift) { return shift == 0.0f ? 8.0f : 4.0f; }

// Where chunk c (eight values, 16 bytes) of row r of a stage lies in its row of
// 4 KS chunks: the rows of one read (16 adjacent ones, at the same columns) lie
// on different banks.
template <int KS>
EP_DEV int front_chunk(int r, int c)
{
    return c ^ (KS == 4 ? r & 15 : KS == 3 ? (r >> 2) & 3 : (r >> 1) & 7);
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));

// 16 bytes a lane from offset `off` of the `bytes` at p (past them: zeros) to the
// lane's place among 64 x 16 adjacent bytes of LDS.
EP_DEV void lds_rows(const void *p, uint32_t bytes, uint16_t *lds, int off)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_rsrc(p, bytes), (__attribute__((address_space(3))) void *)lds, 16, off, 0, 0, 0);
}

// Output columns a lane that attend_kernel.h takes for heads of up to 32 KS values.
constexpr int front_columns(int KS) { return KS == 2 ? 4 : 8; }

// A workgroup's two stages: keys, then values.  They are arrays of their own: the
// compiler waits for rows on their way into an array before it reads from it.
// Where the workgroup is one of attend_body's, it joins its waves' outputs in them.
template <int KS>
struct FrontShared {
    typedef AttendShared<16, 16 * front_columns(KS)> Body;
    static constexpr int kValues = 2 * kFrontStage * 32 * KS, kOutputs = sizeof(typename Body::Outputs) / 2;
    typedef uint16_t Even[kValues > kOutputs ? kValues : kOutputs];
    typedef uint16_t Odd[kValues];
    static EP_DEV Even &even()
    {
        __shared__ __attribute__((aligned(16))) Even s;
        return s;
    }
    static EP_DEV Odd &odd()
    {
        __shared__ __attribute__((aligned(16))) Odd s;
        return s;
    }
    static EP_DEV typename Body::Outputs &outputs() { return *(typename Body::Outputs *)even(); }
    static EP_DEV typename Body::Rows &maxima() { return *(typename Body::Rows *)odd(); }
    static EP_DEV typename Body::Rows &sums() { return *(typename Body::Rows *)(odd() + 1024); }
    static EP_DEV typename Body::Positions &positions() { return *(typename Body::Positions *)(odd() + 2048); }
};

template <typename QOP, int CODE, int KS>
EP_DEV void front_body(const FrontArgs &a, uint32_t at)
{
    constexpr bool k8 = CODE == EP_I8 || CODE == EP_E4M3;
    constexpr int ES = k8 ? 1 : 2, NC = 2 * KS, DM = 32 * KS, TP = kFrontStage, NT = TP / 16;
    constexpr int NK = KS;           // chunks of a stage's keys, and of its values, that a lane brings
    using VOP = typename std::conditional<k8, OpBf16, QOP>::type;
    auto &s_even = FrontShared<KS>::even();
    auto &s_odd = FrontShared<KS>::odd();
    __shared__ float s_ks[2][k8 ? TP : 1], s_vs[2][k8 ? TP : 1];
    __shared__ int s_id[2][kFrontWaves], s_lo[4], s_hi[4];     // page ids of the stages, 16 positions each

    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int H = a.c.heads, D = a.c.D;
    const float nan = __uint_as_float(0x7fc00000u);
    // Workgroups go to the eight XCDs in turn: those that read one piece of one
    // head (its row groups) share an XCD's L2.
    const uint32_t pairs = (uint32_t)H * a.splits;
    uint32_t pair, group;
    {
        const uint32_t x = at & 7, y = at >> 3;
        pair = (y / a.groups) * 8 + x;
        group = y % a.groups;
    }
    if (pair >= pairs)
        return;
    const int h = pair % (uint32_t)H, split = pair / (uint32_t)H;
    const int row0 = group * kFrontRows + 32 * wave, row_end = a.rows;

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
    if (lane == 0) {
        s_lo[wave] = lo;
        s_hi[wave] = hi;
    }
    __syncthreads();
    const int all_lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3])), all_hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
    // stages that the group's rows reach, this piece's share of them
    int j = 0, count = 0;
    if (all_hi >= 0) {
        const int j0 = all_lo / TP, stages = all_hi / TP + 1 - j0;
        j = j0 + (int)((int64_t)stages * split / a.splits);
        count = j0 + (int)((int64_t)stages * (split + 1) / a.splits) - j;
    }
    // any page of these that the pool lacks
    int lacks = 0;
    if (count > 0)
        for (int p = (j * TP >> a.c.page_shift) + tid; p <= (min((j + count) * TP, a.limit) - 1) >> a.c.page_shift; p += 64 * kFrontWaves)
            lacks |= a.tok.table[p] < 0 || a.tok.table[p] >= a.c.n_pages;
    const bool any_bad = __syncthreads_or(lacks);

    // ---- staging
    uint2 kr[k8 ? NK : 1], vr[k8 ? NK : 1];
    float sr[2];
    auto stage = [&](auto odd) -> uint16_t * {
        if constexpr (decltype(odd)::value)
            return s_odd;
        else
            return s_even;
    };
    // A wave brings 16 adjacent rows of each stage, which lie on one page: their
    // descriptor is the wave's, a lane's place in them the same on every stage.
    static_assert(NK * 64 == 16 * 4 * KS, "sixteen rows a wave");
    int off[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const int x = 64 * i + lane, r = x / (4 * KS), c = front_chunk<KS>(r, x % (4 * KS));
        off[i] = 8 * c < D ? (r * D + 8 * c) * ES : kAttOut;
    }
    // Id of the page that the wave's rows of stage j lie on.
    auto page_of = [&](int j) { return a.tok.table[min(j * TP + 16 * wave, a.limit - 1) >> a.c.page_shift]; };
    // Their first row in the pool; -1: past the limit, or not there
    auto row_of = [&](int j, int id) -> int64_t {
        const int p = j * TP + 16 * wave;
        return p < a.limit && id >= 0 && id < a.c.n_pages ? ((int64_t)id * H + h) * a.c.page + (p & (a.c.page - 1)) : -1;
    };
    // The wave's rows of `pool` from `row`: into dst, or (8 bits) into regs.
    auto load_rows = [&](int64_t row, const void *pool, uint16_t *dst, uint2 *regs) {
        const char *src = (const char *)pool + (row < 0 ? 0 : row * (D * ES));
        const uint32_t bytes = row < 0 ? 0u : 16u * D * ES;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            if constexpr (k8) {
                const auto w = __builtin_amdgcn_raw_buffer_load_b64(buffer_rsrc(src, bytes), off[i], 0, 0);
                regs[i] = make_uint2(w[0], w[1]);
            } else      // lane l writes 16 bytes at 16 l from there
                lds_rows(src, bytes, &dst[8 * (64 * (NK * wave + i))], off[i]);
        }
    };
    auto load_scales = [&](int64_t row) {
        if constexpr (k8) {
            const uint32_t bytes = row < 0 ? 0u : 64u;
            const int64_t at = row < 0 ? 0 : row;
            sr[0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buffer_rsrc(a.c.k_scale + at, bytes), 4 * n, 0, 0));
            sr[1] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buffer_rsrc(a.c.v_scale + at, bytes), 4 * n, 0, 0));
        }
    };

    // ---- the running softmax
    constexpr float kSlack = front_slack(VOP::kShift), kShift = VOP::kShift == 0.0f ? 0.0f : VOP::kShift - kSlack;
    float m[2], l[2];
    f32x4_t o[2][NC];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        m[mt] = -INFINITY;
        l[mt] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            o[mt][c] = (f32x4_t){0, 0, 0, 0};
    }
    f32x4_t sc[2][NT];               // scores of the stage at hand
    u32x4_t ph[2][NT / 2], pl[2][NT / 2];       // its weights, in two terms
    int at0 = 0;                     // its first position
    bool some = false;               // any row sees any of it

    auto scores = [&](auto odd, int j) {
        at0 = j * TP;
        some = at0 <= hi && at0 + TP > lo;
        if (!some)
            return;
        const uint16_t *const src = stage(odd);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            sc[0][t] = sc[1][t] = (f32x4_t){0, 0, 0, 0};
            const int r = 16 * t + n;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const u32x4_t f = *(const u32x4_t *)&src[r * DM + 8 * front_chunk<KS>(r, 4 * k + g)];
                sc[0][t] = QOP::mfma(f, q[0][k], sc[0][t]);
                sc[1][t] = QOP::mfma(f, q[1][k], sc[1][t]);
            }
        }
    };
    // Bit e: row (mt, n) sees position 16 (e / 4) + 4 g + e % 4 of the stage at hand.
    auto seen_by = [&](int mt) {
        uint32_t seen = 0;
#pragma unroll
        for (int e = 0; e < 4 * NT; ++e) {
            const int p = at0 + 16 * (e / 4) + 4 * g + e % 4;
            seen |= (uint32_t)(p >= first[mt] && p <= last[mt]) << e;
        }
        return seen;
    };
    auto softmax = [&](auto cuts, auto odd) {
        constexpr bool cut = decltype(cuts)::value;
        if (!some)
            return;
        float vs[k8 ? 4 * NT : 1];
        if constexpr (k8) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4_t ks;
                __builtin_memcpy(&ks, __builtin_assume_aligned(&s_ks[decltype(odd)::value][16 * t + 4 * g], 16), 16);
                __builtin_memcpy(vs + 4 * t, __builtin_assume_aligned(&s_vs[decltype(odd)::value][16 * t + 4 * g], 16), 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ks[i] *= a.scale;
                    sc[0][t][i] *= ks[i];
                    sc[1][t][i] *= ks[i];
                }
            }
        } else
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sc[mt][t][i] *= a.scale;
        if constexpr (cut)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int id = s_id[decltype(odd)::value][t];
                const bool bad = id < 0 || id >= a.c.n_pages;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = at0 + 16 * t + 4 * g + i;
                        sc[mt][t][i] = !(p >= first[mt] && p <= last[mt]) ? -INFINITY : bad ? nan : sc[mt][t][i];
                    }
            }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            float top = sc[mt][0][0];
#pragma unroll
            for (int e = 1; e < 4 * NT; ++e)
                top = fmaxf(top, sc[mt][e / 4][e % 4]);
            top = fmaxf(m[mt], xor32_max(xor16_max(top)));
            if (__any(top > m[mt] + kSlack)) {
                const float base = top == -INFINITY ? 0.0f : top;
                const float keep = __builtin_amdgcn_exp2f(m[mt] - base);
                l[mt] *= keep;
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[mt][c][i] *= keep;
                m[mt] = top;
            }
            const float base = m[mt] == -INFINITY ? 0.0f : m[mt];
            const uint32_t seen = k8 && cut ? seen_by(mt) : 0u;
#pragma unroll
            for (int e = 0; e < 4 * NT; e += 2) {
                float w[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    w[x] = sc[mt][e / 4][e % 4 + x] - base;
                    if constexpr (kShift != 0.0f)
                        w[x] += kShift;          // on the difference: a score past 2^24 would round it away
                    w[x] = __builtin_amdgcn_exp2f(w[x]);
                    l[mt] += w[x];
                    if constexpr (k8)
                        w[x] = cut && !(seen >> (e + x) & 1) ? 0.0f : w[x] * vs[e + x];
                }
                const uint32_t h2 = VOP::pack(w[0], w[1]);
                ph[mt][e / 8][e / 2 % 4] = h2;
                pl[mt][e / 8][e / 2 % 4] = VOP::pack(w[0] - VOP::low(h2), w[1] - VOP::high(h2));
            }
        }
    };
    // Values 16 c + n of positions 4 g + i, and of those 16 behind, from row r0 of
    // the stage: a lane names a quarter of row n / 4 of its four.
    auto column = [&](auto odd, int r0, int c) {
        uint16_t *const src = stage(odd) + TP * DM;
        u32x4_t f;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = r0 + 16 * t + 4 * g + n / 4;
            const s16x4_t w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4_t *)&src[r * DM + 8 * front_chunk<KS>(r, 2 * c + (n >> 1 & 1)) + 4 * (n & 1)]);
            uint2 u;
            __builtin_memcpy(&u, &w, 8);
            f[2 * t] = u.x;
            f[2 * t + 1] = u.y;
        }
        return f;
    };
    auto sums = [&](auto cuts, auto odd) {
        if (!some)
            return;
        if constexpr (!decltype(cuts)::value)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int u = 0; u < NT / 2; ++u) {
                    const u32x4_t f = column(odd, 32 * u, c);
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
                        o[mt][c] = VOP::mfma(f, pl[mt][u], VOP::mfma(f, ph[mt][u], o[mt][c]));
                }
        // Values that no row sees become zero; what some rows see and others not
        // is taken out if it is not finite, and added where it is seen.
        if constexpr (decltype(cuts)::value)
#pragma unroll
            for (int u = 0; u < NT / 2; ++u) {
                u32x4_t keep, one[2];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int p = at0 + 32 * u + 16 * (e / 2) + 4 * g + 2 * (e % 2);
                    keep[e] = (p >= lo && p <= hi ? 0xffffu : 0u) | (p + 1 >= lo && p + 1 <= hi ? 0xffff0000u : 0u);
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
                        one[mt][e] = (p >= first[mt] && p <= last[mt] ? VOP::kOne : 0u) |
                                     (p + 1 >= first[mt] && p + 1 <= last[mt] ? VOP::kOne << 16 : 0u);
                }
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    __builtin_amdgcn_sched_barrier(0);       // a column's registers at a time
                    u32x4_t f = column(odd, 32 * u, c), bad;
                    uint32_t any = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f[e] &= keep[e];
                        bad[e] = CODE == EP_I8 || !ragged ? 0u : not_finite<VOP::kDtype>(f[e]);
                        any |= bad[e];
                        f[e] &= ~bad[e];
                        bad[e] &= VOP::kOne | VOP::kOne << 16;
                    }
                    if (CODE != EP_I8 && __any(any != 0))
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt) {
                            const f32x4_t hits = VOP::mfma(bad, one[mt], (f32x4_t){0, 0, 0, 0});
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                o[mt][c][i] = hits[i] > 0.0f ? nan : o[mt][c][i];
                        }
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
                        o[mt][c] = VOP::mfma(f, pl[mt][u], VOP::mfma(f, ph[mt][u], o[mt][c]));
                }
            }
    };

    // ---- stages: one is multiplied, the next is on its way
    const auto even = std::false_type();
    const auto odd = std::true_type();
    int id = 0, next_id = 0;         // pages of the wave's rows of the next stage, and of the one after it
    auto begin_rows = [&](auto is_odd, int j) {
        const int64_t row = row_of(j, id);
        load_rows(row, a.c.k, stage(is_odd), kr);
        load_rows(row, a.c.v, stage(is_odd) + TP * DM, vr);
        load_scales(row);
        if (lane == 0)
            s_id[decltype(is_odd)::value][wave] = id;
    };
    auto end_rows = [&](auto is_odd) {
        if constexpr (k8) {
            uint16_t *const dst = stage(is_odd);
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const int x = 64 * (NK * wave + i) + lane;
                *(u32x4_t *)&dst[8 * x] = decode8<QOP, CODE>(kr[i].x, kr[i].y);
                *(u32x4_t *)&dst[TP * DM + 8 * x] = decode8<VOP, CODE>(vr[i].x, vr[i].y);
            }
            if (lane < 16) {
                s_ks[decltype(is_odd)::value][16 * wave + lane] = sr[0];
                s_vs[decltype(is_odd)::value][16 * wave + lane] = sr[1];
            }
        }
    };
    auto turn = [&](auto cuts, auto is_odd, int x) {
        const std::integral_constant<bool, !decltype(is_odd)::value> other;
        // With no branch around it (behind the last stage there are no rows): the
        // compiler forgets at a branch's end which loads go to which array.
        id = x + 1 < count ? __builtin_amdgcn_readfirstlane(next_id) : -1;
        begin_rows(other, j + x + 1);
        next_id = page_of(j + x + 2);
        scores(is_odd, j + x);
        softmax(cuts, is_odd);
        // what looks for values that are not finite takes the registers of the rows on their way
        if (decltype(cuts)::value)
            end_rows(other);
        sums(cuts, is_odd);
        if (!decltype(cuts)::value)
            end_rows(other);
        __syncthreads();             // the next stage is there, and this one's readers are done
    };
    if (count > 0) {
        if (D < DM) {        // places that no load reaches
            for (int x = tid; x < 2 * TP * DM / 8; x += 64 * kFrontWaves) {
                *(u32x4_t *)&s_even[8 * x] = (u32x4_t){0, 0, 0, 0};
                *(u32x4_t *)&s_odd[8 * x] = (u32x4_t){0, 0, 0, 0};
            }
            __syncthreads();
        }
        id = __builtin_amdgcn_readfirstlane(page_of(j));
        next_id = page_of(j + 1);
        begin_rows(even, j);
        end_rows(even);
        __syncthreads();
        auto turns = [&](auto cuts) {
            for (int x = 0;; x += 2) {
                turn(cuts, even, x);
                if (x + 1 >= count)
                    break;
                turn(cuts, odd, x + 1);
                if (x + 2 >= count)
                    break;
            }
        };
        // Scores are masked one by one where a row of the wave sees a part of
        // the piece only, or a page is missing: in a loop of its own (branches in
        // one had the compiler keep the sums twice).
        if (j * TP < in_lo || (j + count) * TP - 1 > in_hi || any_bad)
            turns(std::true_type());
        else
            turns(std::false_type());
    }

    // ---- the piece's part
    const int64_t slot = ((int64_t)group * H + h) * a.splits + split;
    // weights of the other kernels' parts are 2^kShift, without the slack
    constexpr float up = VOP::kShift == 0.0f ? 1.0f : (float)(1 << (int)kSlack);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        l[mt] = xor32_sum(xor16_sum(l[mt]));
        const int r = 32 * wave + 16 * mt + n;
        if (group * kFrontRows + r >= row_end)
            continue;
        const int64_t at = slot * kFrontRows + r;
        if (g == 0)
            a.part_ml[at] = make_float2(m[mt], l[mt] * up);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            f32x4_t z;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                z[i] = o[mt][c][i] * up;
            if (16 * c < D)
                *(f32x4_t *)(a.part_o + at * D + 16 * c + 4 * g) = z;
        }
    }
}

template <typename QOP, int CODE, int KS>
__global__ void __launch_bounds__(64 * kFrontWaves, kFrontOccupancy) front_kernel(FrontArgs a)
{
    front_body<QOP, CODE, KS>(a, a.first_wg + blockIdx.x);
}

// And the sequences' own pages in the same launch (up to kTogetherRows rows of one
// sequence on a cache head, 16 a unit).  The shared pages' workgroups come first and the others where
// those leave room: they wait for memory while the former multiply, and there is
// no end of one launch and beginning of another between them (the calls above:
// 176 -> 157 to 164 us and 91 -> 85; in turns 170 and 117, the others first 163 and 91).
struct FrontTails {
    FrontArgs front;
    AttendParts tails;
    uint32_t fronts;         // workgroups of the former, a multiple of eight
};
template <typename QOP, int CODE, int KS>
__global__ void __launch_bounds__(64 * kFrontWaves, kFrontOccupancy) front_tails_kernel(FrontTails a)
{
    constexpr bool k8 = CODE == EP_I8 || CODE == EP_E4M3;
    if (blockIdx.x < a.fronts)
        front_body<QOP, CODE, KS>(a.front, blockIdx.x);
    else
        attend_body<QOP, CODE, k8 && KS == 3 ? 4 : KS, front_columns(KS), 1, true, FrontShared<KS>>(a.tails, blockIdx.x - a.fronts);
}

template <typename QOP, int CODE>
void front_by_size(const FrontArgs &a, unsigned grid, hipStream_t st)
{
    if (a.c.D <= 64)
        front_kernel<QOP, CODE, 2><<<grid, 64 * kFrontWaves, 0, st>>>(a);
    else if (a.c.D <= 96)
        front_kernel<QOP, CODE, 3><<<grid, 64 * kFrontWaves, 0, st>>>(a);
    else
        front_kernel<QOP, CODE, 4><<<grid, 64 * kFrontWaves, 0, st>>>(a);
}

template <typename QOP, int CODE>
void front_tails_by_size(const FrontTails &a, unsigned grid, hipStream_t st)
{
    if (a.front.c.D <= 64)
        front_tails_kernel<QOP, CODE, 2><<<grid, 64 * kFrontWaves, 0, st>>>(a);
    else if (a.front.c.D <= 96)
        front_tails_kernel<QOP, CODE, 3><<<grid, 64 * kFrontWaves, 0, st>>>(a);
    else
        front_tails_kernel<QOP, CODE, 4><<<grid, 64 * kFrontWaves, 0, st>>>(a);
}

void attend_front_tails(const FrontTails &a, int q_dtype, unsigned grid, hipStream_t st);
void attend_front(const FrontArgs &a, int q_dtype, unsigned grid, hipStream_t st);

}  // namespace ep
