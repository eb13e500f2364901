// Attention of new tokens over a paged key-value cache: the kernel template
// (attend.hip plans and joins; attend_gen_*.hip instantiate).
//
//   out[r] = sum_j softmax_j(scale q[r] . k[j]) v[j],   first(r) <= j <= last(r)
//
// The rows of one matrix tile are the query heads that share a cache head,
// over all new tokens of a sequence (a "unit" is up to 16 MT of them); a
// segment is one unit on one cache head, cut into tiles of 32 positions.
//
// A wave takes whole tiles straight from memory to registers, with nothing
// exchanged between lanes on the way:
//   S^T = K Q^T: lane (n = lane & 15, g = lane >> 4) gives key row 16 t + n,
//     values 8 g .. 8 g + 7 of each 32 (8-bit caches: 16 g .. of each 64,
//     taken as two steps), and gets the scores of positions
//     16 t + 4 g + i of query row n.
//   O^T = V^T P^T: that is the layout of the second product's B operand if
//     its k index 8 g + 4 t + i means position 16 t + 4 g + i.  The A operand
//     then wants, for output n, eight positions of one column: lane n takes
//     CW adjacent columns of those eight rows (16 lanes read one whole row),
//     and the CW products of columns CW n + t, t = 0 .. CW - 1, need only the
//     16-bit halves of two rows put side by side.
// A row's maximum, sum and output live in the four lanes of one n, so the
// running softmax costs two lane exchanges a tile.
//
// Rounding: scores, softmax and sums are f32; the weights enter the second
// product as two 16-bit terms (w and what its rounding lost), which leaves
// 2^-16 of each where one term would leave 2^-8 (bf16), for 1 - 2% of the time
// (8% with 64 rows a key head in int8).  8-bit codes are exact in either 16-bit
// type; their scales multiply scores and weights.  In f16 the weights are
// 2^15 exp(s - max), so that a long tail of small ones stays above f16's least
// number.  An infinity among the values that a row sees gives it an infinity
// or a NaN (it meets both terms).
//
// Bound by the bytes of keys and values: 4 x 131072 positions of 8 heads of
// 128 in bf16, 2.06 GB, take 297 us (6.9 TB/s) and 48 of up to 8192 in int8,
// 441 MB, 81 us, four waves a workgroup with a tile of 16 KiB (bf16) in flight
// each, one or two workgroups a compute unit.  Short calls are a chain of loads:
// arguments, positions with pages and queries, keys and values, 7 us in all for
// 129 positions; the code is kept small (10 KB) because it is fetched cold.
#pragma once

#include "ep_common.h"
#include "ep_internal.h"
#include "ep_paged.h"

namespace ep {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kAttTile = 32;             // positions a wave takes at a time
constexpr int kAttWaves = 4;             // waves of a workgroup: they take tiles in turn
constexpr int kAttOnce = 2;              // a load's non-temporal bit: rows that are read once
constexpr int kAttOut = 0x40000000;      // an offset past every descriptor below: reads zeros

struct AttendArgs {
    const void *q;
    int64_t q_sb, q_ss, q_sh;
    PagedTokens tok;
    PagedCache c;
    float scale;             // of the scores, times log2(e)
    int window;              // 1 .. cap
    int cap;                 // positions that the table has pages for
    void *out;
    int G, rows;             // query heads a cache head; rows of a sequence on one cache head (S G)
    int blocks;              // units of a sequence
    uint32_t units;
    uint32_t first_wg;       // of this launch, where a call takes more workgroups than one launch can have
    int workers;             // workgroups that share all tiles evenly; 0: one workgroup a segment
    int few;                 // shares of a large call, of more than 16 tiles each
    int piece;               // tiles' time that beginning and ending a piece takes
    int keys_once;           // keys are loaded past the caches, as values are
    int slot_rows;           // rows kept of a piece: min(rows, 16 MT)
    int2 *desc;              // [segments]: first slot, pieces
    float2 *part_ml;         // [2 workers][slot_rows]: maximum, sum
    float *part_o;           // [2 workers][slot_rows][D]
};

// What a call's units, rows and positions are:
//   kWhole: a unit is up to 16 MT rows of one sequence, which see its pages
//     from position 0 on (the pieces' outputs join where there are several);
//   kParts: the tables' first `shared` pages are those of sequence 0.  The
//     first `front` units are rows of the whole batch, over those pages; the
//     rest is as in kWhole, over the pages behind them, positions counted
//     from there.  Every output stays a part: the join adds them up (where the
//     shared pages go through LDS, through_lds() of attend.hip, they are
//     attend_front.h's and there are no such units);
//   kBlocks: a unit is up to 16 rows of one token, and tile after tile goes
//     over the `take` pages that a list names for it, in `cuts` equal pieces
//     (8 tokens of 64 pages of 64 positions, 8 heads of 128 in bf16, 134 MB: 23 us).
enum AttendMode { kWhole, kParts, kBlocks };

struct AttendWhole : AttendArgs {
    static constexpr AttendMode kMode = kWhole;
};
struct AttendParts : AttendArgs {
    static constexpr AttendMode kMode = kParts;
    int front, front_rows;   // units over the shared pages; query rows of the batch on one cache head
    int shared, from;        // pages, and positions in them
    int front_splits;        // front 0: pieces that attend_front.h cut the shared positions into,
    int64_t front_at;        // and where they begin among the parts' rows
};
struct AttendBlocks : AttendArgs {
    static constexpr AttendMode kMode = kBlocks;
    const int32_t *list;     // [B][S][heads][take]
    int take, cuts;
};

// v, computed anew where it is used: what follows from it is not kept in
// registers across the loops.
EP_DEV int opaque(int v)
{
    asm volatile("" : "+v"(v));
    return v;
}

EP_DEV int dpp_row_max(int v)
{
    const auto step = [&](int o) { v = v > o ? v : o; };
    step(__builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x124, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false));
    return __builtin_amdgcn_readfirstlane(v);
}

// Position of token (b, s): in [0, cap), -1 for padding, cap past the table.
EP_DEV int attend_position(const AttendArgs &a, int64_t b, int s)
{
    const int64_t p = a.tok.pos[b * a.tok.pos_sb + s * a.tok.pos_ss];
    return p < 0 ? -1 : p >= a.cap ? a.cap : (int)p;
}

EP_DEV int first_seen(const AttendArgs &a, int p) { return p >= a.window ? p - a.window + 1 : 0; }

// A unit: its first row and how many rows it counts among, the token of row 0,
// the sequence whose table it reads, and the positions [from, limit) of it.
struct AttendUnit {
    int r0, rows;
    int64_t b, t0;
    int from, limit;
};
template <int RM, typename ARGS>
EP_DEV AttendUnit attend_unit(const ARGS &a, uint32_t u)
{
    if constexpr (ARGS::kMode == kParts) {
        if (u < (uint32_t)a.front)
            return {(int)u * RM, a.front_rows, 0, 0, 0, a.from};
        u -= a.front;
    }
    const uint32_t b = u / (uint32_t)a.blocks;
    const int r0 = (int)(u - b * a.blocks) * RM;
    if constexpr (ARGS::kMode == kBlocks)
        return {r0, a.G, b / (uint32_t)a.tok.S, b, 0, a.cap};
    else if constexpr (ARGS::kMode == kParts)
        return {r0, a.rows, b, (int64_t)b * a.tok.S, a.from, a.cap - a.from};
    else
        return {r0, a.rows, b, 0, 0, a.cap};
}

// Token (b, s) of row `row` of a unit; its tokens count from that of row 0.
struct AttendToken {
    int64_t b;
    int s, head;     // head: within the group
};
template <typename ARGS>
EP_DEV AttendToken attend_token_at(const ARGS &a, const AttendUnit &u, int t, int head)
{
    if constexpr (ARGS::kMode == kWhole)
        return {u.b, t, head};
    else {
        const uint32_t at = (uint32_t)(u.t0 + t), b = at / (uint32_t)a.tok.S;
        return {b, (int)(at - b * (uint32_t)a.tok.S), head};
    }
}
template <typename ARGS>
EP_DEV AttendToken attend_token(const ARGS &a, const AttendUnit &u, int row)
{
    const int t = (uint32_t)row / (uint32_t)a.G;
    return attend_token_at(a, u, t, row - t * a.G);
}

// What a row at position p sees of its unit's positions, counted from the
// unit's first; false: nothing.
template <typename ARGS>
EP_DEV bool attend_span(const ARGS &a, const AttendUnit &u, int p, int &first, int &last)
{
    bool some = p >= 0 && p < a.cap;
    first = first_seen(a, p);
    last = p;
    if constexpr (ARGS::kMode == kParts) {
        first = max(first - u.from, 0);
        last = min(p - u.from, u.limit - 1);
        some = some && first <= last;
    }
    first = some ? first : a.cap;
    last = some ? last : -1;
    return some;
}

// Tiles that the rows of unit u reach (one at least: its outputs are written
// with that tile), and the first of them.
template <int RM, typename ARGS>
EP_DEV uint32_t unit_tiles(const ARGS &a, uint32_t u, uint32_t &first)
{
    const AttendUnit unit = attend_unit<RM>(a, u);
    const int r0 = unit.r0, r1 = min(r0 + RM, unit.rows);
    const int s0 = (uint32_t)r0 / (uint32_t)a.G, s1 = (uint32_t)(r1 - 1) / (uint32_t)a.G;
    int lo = a.cap, hi = -1;
    for (int s = s0; s <= s1; s += 4) {
        int p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {    // four loads in flight; the last token again past the end
            const AttendToken t = attend_token_at(a, unit, min(s + i, s1), 0);
            p[i] = attend_position(a, t.b, t.s);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int f, l;
            if (attend_span(a, unit, p[i], f, l)) {
                hi = max(hi, l);
                lo = min(lo, f);
            }
        }
    }
    first = hi < 0 ? 0u : (uint32_t)(lo / kAttTile);
    return hi < 0 ? 1u : (uint32_t)(hi / kAttTile) - first + 1;
}

// 16-bit arithmetic of a product's operands.
struct OpBf16 {
    static constexpr int kDtype = EP_BF16;
    static constexpr float kShift = 0.0f;
    static constexpr uint32_t kOne = 0x3f80u;
    static EP_DEV f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c)
    {
        bf16x8_t x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    }
    // Two values rounded to 16 bits, and the rest of each rounded likewise.
    static EP_DEV uint32_t pack(float x, float y)
    {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        const bf16x2_t h = __builtin_convertvector((f32x2_t){x, y}, bf16x2_t);
        uint32_t u;
        __builtin_memcpy(&u, &h, 4);
        return u;
    }
    static EP_DEV float low(uint32_t u) { return __uint_as_float(u << 16); }
    static EP_DEV float high(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
};
struct OpF16 {
    static constexpr int kDtype = EP_F16;
    static constexpr float kShift = 15.0f;
    static constexpr uint32_t kOne = 0x3c00u;
    static EP_DEV f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c)
    {
        f16x8_t x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    }
    static EP_DEV uint32_t pack(float x, float y)
    {
        const f16x2_t h = {(f16_t)x, (f16_t)y};
        uint32_t u;
        __builtin_memcpy(&u, &h, 4);
        return u;
    }
    static EP_DEV float low(uint32_t u) { return (float)as_f16x2(u)[0]; }
    static EP_DEV float high(uint32_t u) { return (float)as_f16x2(u)[1]; }
};

// Two 8-bit codes of w (bytes B, B + 1 with HI = B / 2) as f32.
template <int CODE, bool HI>
EP_DEV void codes2(uint32_t w, float &x, float &y)
{
    if constexpr (CODE == EP_I8) {
        x = (float)(int8_t)(w >> (HI ? 16 : 0));
        y = (float)(int8_t)(w >> (HI ? 24 : 8));
    } else {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        const f32x2_t v = __builtin_amdgcn_cvt_pk_f32_fp8(w, HI);
        x = v[0];
        y = v[1];
    }
}

// All bits set in each value of w that is infinite or NaN.
template <int CODE>
EP_DEV uint32_t not_finite(uint32_t w)
{
    if constexpr (CODE == EP_E4M3) {     // NaN: 0x7f; one more sets the sign bit
        const uint32_t h = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        return (h >> 7) * 0xffu;
    } else {                             // all exponent bits; one more of them sets the sign bit
        constexpr uint32_t e = CODE == EP_BF16 ? 0x7f807f80u : 0x7c007c00u, one = CODE == EP_BF16 ? 0x00800080u : 0x04000400u;
        const uint32_t h = ((w & e) + one) & 0x80008000u;
        return (h >> 15) * 0xffffu;
    }
}

// The upper halves of two f32 side by side: codes are exact in bf16.
EP_DEV uint32_t high_halves(float x, float y)
{
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}

// Eight codes as an operand.
template <typename OP, int CODE>
EP_DEV u32x4_t decode8(uint32_t w0, uint32_t w1)
{
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x, y;
        if (i & 1)
            codes2<CODE, true>(i < 2 ? w0 : w1, x, y);
        else
            codes2<CODE, false>(i < 2 ? w0 : w1, x, y);
        if constexpr (OP::kDtype == EP_BF16)
            r[i] = high_halves(x, y);
        else
            r[i] = OP::pack(x, y);
    }
    return r;
}

EP_DEV __amdgpu_buffer_rsrc_t tile_rsrc(const void *base, int64_t byte, bool ok, int bytes)
{
    return buffer_rsrc((const char *)base + (ok ? byte : 0), ok ? (uint32_t)bytes : 0u);
}

// Workgroups of a kernel that a compute unit holds (waves of a SIMD).  Three of
// the one-token kernels would fit at 128 values, and gain nothing.  `lookout`:
// several tokens over values that may each be infinite or a NaN; what looks
// for them takes some 40 registers, too many for two waves with 12 columns
// (33 would go through memory).
constexpr int attend_occupancy(int CW, int MT, bool lookout)
{
    return CW == 4 ? (MT == 1 ? 3 : 2) : CW == 8 || (CW == 12 && MT == 1 && !lookout) ? 2 : 1;
}

// Output columns a lane for heads of D values: 16 lanes read a row, and a
// lane's columns end where the row does.  Against 16, 12 columns leave room for
// a second wave on the SIMD with one new token, and a quarter of the second
// product out (16 x 2-4 thousand positions: 144 int8 values 23.3 us, 27.0 with
// 16 columns; 192 bf16 values 36.8 and 37.8, 32 rows a key head 45.8 and 48.7).
constexpr int attend_columns(int D) { return D <= 64 ? 4 : D <= 128 ? 8 : D <= 192 && D % 12 == 0 ? 12 : 16; }

// What a workgroup joins its waves' outputs by: outputs, maxima and sums, the
// rows' positions.
template <int RM, int DP>
struct AttendShared {
    typedef float Outputs[kAttWaves][RM][DP + 4];
    typedef float Rows[kAttWaves][RM];
    typedef int Positions[RM];
    static EP_DEV Outputs &outputs()
    {
        __shared__ Outputs s;
        return s;
    }
    static EP_DEV Rows &maxima()
    {
        __shared__ Rows s;
        return s;
    }
    static EP_DEV Rows &sums()
    {
        __shared__ Rows s;
        return s;
    }
    static EP_DEV Positions &positions()
    {
        __shared__ Positions s;
        return s;
    }
};

// wg: the workgroup's number, of those that this body is for.
// QOP: type of the queries; CODE: EP_I8, EP_E4M3, or QOP's type.  KS: steps of
// 32 values of a head, CW: output columns a lane (16 CW >= D), MT: 16-row
// tiles of query rows.  RAGGED: rows of a unit may differ in what they see.
template <typename QOP, int CODE, int KS, int CW, int MT, bool RAGGED, typename SHARED = AttendShared<16 * MT, 16 * CW>, typename ARGS>
EP_DEV void attend_body(const ARGS &a, uint32_t wg)
{
    constexpr AttendMode MODE = ARGS::kMode;
    constexpr bool k8 = CODE == EP_I8 || CODE == EP_E4M3;
    constexpr int ES = k8 ? 1 : 2, KL = k8 ? KS / 2 : KS, RM = 16 * MT, DP = 16 * CW, VW = CW * ES / 4;
    static_assert(!k8 || KS % 2 == 0, "8-bit keys are read in chunks of two steps");
    using VOP = typename std::conditional<k8, OpBf16, QOP>::type;
    auto &s_o = SHARED::outputs();
    auto &s_m = SHARED::maxima();
    auto &s_l = SHARED::sums();
    auto &s_p = SHARED::positions();
    // Queries of more than one row tile stay in LDS: their registers are what
    // a second wave on the SIMD needs.
    constexpr bool kQueriesInLds = MT > 1;
    __shared__ u32x4_t s_q[kQueriesInLds ? MT * KS * 64 : 1];

    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int H = a.c.heads, D = a.c.D;
    const float nan = __uint_as_float(0x7fc00000u);

    // Offsets of this lane's key chunks and value rows within half a tile.
    int koff[2], voff[4];
    const int kbase = n * D * ES + 16 * g;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = (KL - 2 + i) * (k8 ? 64 : 32) + g * (k8 ? 16 : 8);
        koff[i] = d < D ? kbase + (KL - 2 + i) * 64 : kAttOut;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        voff[i] = CW * n < D ? ((4 * g + i) * D + CW * n) * ES : kAttOut;

    // ---- one piece: tiles [t0, t1) of the positions; t0 < 0: all that the
    // unit's rows reach.  slot < 0: the outputs are written.
    auto piece = [&](uint32_t u, int h, int t0, int t1, int slot) {
        const AttendUnit unit = attend_unit<RM>(a, u);
        const int r0 = unit.r0;
        const int lx = opaque(lane), ln = lx & 15, lg = lx >> 4;
        const int32_t *table = a.tok.table + unit.b * a.tok.table_stride;
        int64_t width = a.tok.width;     // pages of this unit's table
        if constexpr (MODE == kParts)
            if (unit.from) {
                table += a.shared;
                width -= a.shared;
            }
        // kBlocks: the page in the list that half (lane & 1) of tile j lies in, -1: none
        auto load_block = [&](int j) {
            if constexpr (MODE == kBlocks) {
                const int32_t *list = a.list + (unit.t0 * H + h) * a.take;
                const int at = (j * kAttTile + 16 * (lane & 1)) >> a.c.page_shift;
                const int block = list[min(at, a.take - 1)];
                return at < a.take && block >= 0 && block < width ? block : -1;
            }
            return 0;
        };
        auto load_ids = [&](int j, int block) {
            const int64_t at = MODE == kBlocks ? block : (int64_t)(j * kAttTile + 16 * (lane & 1)) >> a.c.page_shift;
            return width > 0 ? table[at < 0 ? 0 : at < width ? at : width - 1] : -1;
        };
        // Pages, positions and queries load together where the first tile is
        // known: a share's piece, or no window.
        const bool known = t0 >= 0 || a.window >= a.cap;
        int j = max(t0, 0) + wave, ids = 0, block = 0;
        if (known) {
            block = load_block(j);
            ids = load_ids(j, block);
        }
        int pos[MT], first[MT], last[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int row = r0 + 16 * mt + ln;
            pos[mt] = -1;
            if (row < unit.rows) {
                const AttendToken t = attend_token(a, unit, row);
                pos[mt] = attend_position(a, t.b, t.s);
            }
        }
        __builtin_amdgcn_sched_barrier(0);       // loads return in order: the positions' wait must not cover the queries
        // (mt, k): values of step k of row n, zero past D
        auto query = [&](int mt, int k) {
            const AttendToken t = attend_token(a, unit, min(r0 + 16 * mt + ln, unit.rows - 1));
            const int d = k8 ? 64 * (k / 2) + 16 * lg + 8 * (k & 1) : 32 * k + 8 * lg;
            const int64_t at = t.b * a.q_sb + t.s * a.q_ss + (int64_t)(h * a.G + t.head) * a.q_sh + (d < D ? d : 0);
            return *(const u32x4_t *)((const char *)a.q + 2 * at);
        };
        auto in_head = [&](int k, u32x4_t w) {
            const int d = k8 ? 64 * (k / 2) + 16 * lg + 8 * (k & 1) : 32 * k + 8 * lg;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = d < D ? w[i] : 0u;
            return w;
        };
        constexpr int QN = kQueriesInLds ? (MT * KS + kAttWaves - 1) / kAttWaves : MT * KS;
        u32x4_t q[QN];
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int f = kQueriesInLds ? min(kAttWaves * i + wave, MT * KS - 1) : i;
            q[i] = query(f / KS, f % KS);
        }
        __builtin_amdgcn_sched_barrier(0);
        int lo = -a.cap, hi = -1, in_lo = 0, in_hi = -a.cap;     // over the rows: seen by any (lo negated), by all
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int p = pos[mt];
            const bool some = attend_span(a, unit, p, first[mt], last[mt]);
            lo = max(lo, some ? -first[mt] : -a.cap);
            hi = max(hi, last[mt]);
            // kParts: a row that sees nothing here masks every tile (a padded one may hold anything)
            in_lo = max(in_lo, some ? first[mt] : MODE == kParts && p >= 0 ? a.cap : 0);
            in_hi = max(in_hi, some ? -last[mt] : -a.cap);
            if (wave == 0 && lg == 0)
                s_p[16 * mt + ln] = p;
        }
        lo = -dpp_row_max(lo);
        hi = dpp_row_max(hi);
        in_lo = dpp_row_max(in_lo);
        in_hi = -dpp_row_max(in_hi);
        const bool ragged = lo != in_lo || hi != in_hi;     // rows differ in what they see
        const int end = t0 >= 0 ? t1 : hi < 0 ? 1 : hi / kAttTile + 1;
        if (!known) {
            j = (hi < 0 ? 0 : lo / kAttTile) + wave;
            block = load_block(j);
            ids = load_ids(j, block);
        }

        // ---- loads
        u32x4_t kr[2][KL];
        uint32_t vr[VW][8];      // [dword of the columns][row]
        float ks[8], vs[8];
        bool good[2];
        int64_t at[2];       // row of each half's first position
        int base[2];         // kBlocks: that position (a.cap: none)
        auto locate = [&](int ids, int block, int j) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int64_t id = __builtin_amdgcn_readlane(ids, t);
                const int row = (j * kAttTile + 16 * t) & (a.c.page - 1);
                good[t] = j < end && id >= 0 && id < a.c.n_pages;
                at[t] = (id * H + h) * a.c.page + row;
                if constexpr (MODE == kBlocks) {
                    const int k = __builtin_amdgcn_readlane(block, t);
                    good[t] = good[t] && k >= 0;
                    base[t] = k < 0 ? a.cap : (k << a.c.page_shift) + row;
                }
            }
        };
        auto load_scales = [&](const float *src, float *out) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const auto w = __builtin_amdgcn_raw_buffer_load_b128(tile_rsrc(src, at[t] * 4, good[t], 64), 16 * g, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    out[4 * t + i] = __uint_as_float(w[i]);
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const auto r = tile_rsrc(a.c.k, at[t] * D * ES, good[t], 16 * D * ES);
                if (a.keys_once)
#pragma unroll
                    for (int k = 0; k < KL; ++k)
                        kr[t][k] = __builtin_amdgcn_raw_buffer_load_b128(
                            r, k >= KL - 2 ? koff[k - (KL - 2)] : kbase + 64 * k, 0, kAttOnce);
                else
#pragma unroll
                    for (int k = 0; k < KL; ++k)
                        kr[t][k] = __builtin_amdgcn_raw_buffer_load_b128(
                            r, k >= KL - 2 ? koff[k - (KL - 2)] : kbase + 64 * k, 0, 0);
            }
            if constexpr (k8)
                load_scales(a.c.k_scale, ks);
        };
        auto load_v = [&]() {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const auto r = tile_rsrc(a.c.v, at[t] * D * ES, good[t], 16 * D * ES);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 4 * t + i;
                    if constexpr (VW == 1)
                        vr[0][row] = __builtin_amdgcn_raw_buffer_load_b32(r, voff[i], 0, kAttOnce);
                    else if constexpr (VW == 2) {
                        const auto w = __builtin_amdgcn_raw_buffer_load_b64(r, voff[i], 0, kAttOnce);
                        vr[0][row] = w[0];
                        vr[1][row] = w[1];
                    } else
#pragma unroll
                        for (int c = 0; c < VW; c += 4) {
                            if (c + 4 <= VW) {
                                const auto w = __builtin_amdgcn_raw_buffer_load_b128(r, voff[i] + 4 * c, 0, kAttOnce);
#pragma unroll
                                for (int x = 0; x < 4; ++x)
                                    vr[c + x][row] = w[x];
                            } else if (c + 3 == VW) {
                                const auto w = __builtin_amdgcn_raw_buffer_load_b96(r, voff[i] + 4 * c, 0, kAttOnce);
#pragma unroll
                                for (int x = 0; x < 3; ++x)
                                    vr[c + x][row] = w[x];
                            } else {
                                const auto w = __builtin_amdgcn_raw_buffer_load_b64(r, voff[i] + 4 * c, 0, kAttOnce);
                                vr[c][row] = w[0];
                                vr[c + 1][row] = w[1];
                            }
                        }
                }
            }
            if constexpr (k8)
                load_scales(a.c.v_scale, vs);
        };

        // ---- the running softmax
        float m[MT], l[MT];
        f32x4_t o[MT][CW];
        // Outputs that a value which is not finite has reached.  Written into the
        // sums where they happen, they hold some 80 registers more in the loop,
        // which with 16 columns a lane and two row tiles does not fit: 36 of them
        // went through memory, in the queue of the rows' loads (16 x 2-4 thousand
        // positions of 256 bf16 values, 32 rows a key head: 73 us, 57 with a bit
        // each, looked at in the end).  With 8 columns the bits cost some 25 more.
        constexpr bool kHitsApart = RAGGED && CODE != EP_I8 && CW >= 12;
        uint32_t hit[MT][2] = {};
        bool named = false;      // kBlocks: a tile held positions that the rows see
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m[mt] = -INFINITY;
            l[mt] = 0.0f;
#pragma unroll
            for (int t = 0; t < CW; ++t)
                o[mt][t] = (f32x4_t){0, 0, 0, 0};
        }
        locate(ids, block, j);
        block = load_block(j + kAttWaves);
        ids = load_ids(j + kAttWaves, block);
        int ahead = load_block(j + 2 * kAttWaves);      // kBlocks: its page id waits for it
        __builtin_amdgcn_sched_barrier(0);
        load_k();
        __builtin_amdgcn_sched_barrier(0);       // loads return in order: the keys' wait must not cover the values
        load_v();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int f = kQueriesInLds ? min(kAttWaves * i + wave, MT * KS - 1) : i;
            q[i] = in_head(f % KS, q[i]);
            if constexpr (kQueriesInLds)
                s_q[64 * f + lx] = q[i];
        }
        if constexpr (kQueriesInLds)
            lds_barrier();
        for (; j < end; j += kAttWaves) {
            if constexpr (kQueriesInLds)
                asm volatile("" ::: "memory");      // the queries are read again for each tile
            // positions of the tile's halves
            const int j0 = MODE == kBlocks ? base[0] : j * kAttTile, j1 = MODE == kBlocks ? base[1] : j0 + 16;
            const bool bad0 = !good[0], bad1 = !good[1];
            if constexpr (MODE == kBlocks)
                named = named || (j0 <= hi && j0 + 15 >= lo) || (j1 <= hi && j1 + 15 >= lo);
            auto position = [&](int e) { return (e < 4 ? j0 : j1) + 4 * g + e % 4; };
            f32x4_t sc[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    sc[mt][t] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    u32x4_t f;
                    if constexpr (k8)
                        f = decode8<QOP, CODE>(kr[t][k / 2][2 * (k & 1)], kr[t][k / 2][2 * (k & 1) + 1]);
                    else
                        f = kr[t][k];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
                        sc[mt][t] = QOP::mfma(f, kQueriesInLds ? s_q[64 * (mt * KS + k) + lane] : q[mt * KS + k], sc[mt][t]);
                }
            float x[MT][8];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[mt][e] = sc[mt][e / 4][e % 4] * (k8 ? ks[e] * a.scale : a.scale);
            // the next tile's keys (none past the end: empty descriptors)
            __builtin_amdgcn_sched_barrier(0);
            locate(ids, block, j + kAttWaves);
            block = ahead;
            ids = load_ids(j + 2 * kAttWaves, block);
            ahead = load_block(j + 3 * kAttWaves);
            load_k();
            __builtin_amdgcn_sched_barrier(0);

            // A tile that some row sees in part (or that names a page the pool
            // lacks: its scores are NaN) masks its scores one by one.
            const bool edge = min(j0, j1) < in_lo || max(j0, j1) + 15 > in_hi || bad0 || bad1;
            uint32_t seen[MT];
            if (edge) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    seen[mt] = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int p = position(e);
                        const bool in = p >= first[mt] && p <= last[mt];
                        seen[mt] |= (uint32_t)in << e;
                        x[mt][e] = !in ? -INFINITY : (e < 4 ? bad0 : bad1) ? nan : x[mt][e];
                    }
                }
            }
            u32x4_t ph[MT], pl[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
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
                    for (int t = 0; t < CW; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            o[mt][t][i] *= keep;
                }
                m[mt] = top;
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // The shift goes on the difference: on a score past 2^24 it would be
                    // rounded, and the largest weight could pass f16's largest number.
                    w[e] = x[mt][e] - base;
                    if constexpr (VOP::kShift != 0.0f)
                        w[e] += VOP::kShift;
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
            // Values: what no row sees becomes zero (its weights are zero, and
            // zero times a NaN is NaN); what some rows see and others not is
            // taken out if it is not finite, and added where it is seen.
            // Operand of column t: eight rows' values side by side.
            auto column = [&](const uint32_t (&rows)[8], int t) {
                u32x4_t f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (k8) {
                        float v0[2], v1[2];
                        if (t & 2) {
                            codes2<CODE, true>(rows[2 * e], v0[0], v0[1]);
                            codes2<CODE, true>(rows[2 * e + 1], v1[0], v1[1]);
                        } else {
                            codes2<CODE, false>(rows[2 * e], v0[0], v0[1]);
                            codes2<CODE, false>(rows[2 * e + 1], v1[0], v1[1]);
                        }
                        f[e] = high_halves(v0[t & 1], v1[t & 1]);
                    } else {
                        f[e] = __builtin_amdgcn_perm(rows[2 * e + 1], rows[2 * e], t & 1 ? 0x07060302u : 0x05040100u);
                    }
                }
                return f;
            };
            if (edge) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int p = position(r);
                    const uint32_t keep = p >= lo && p <= hi ? ~0u : 0u;
#pragma unroll
                    for (int c = 0; c < VW; ++c)
                        vr[c][r] &= keep;
                }
                if (RAGGED && CODE != EP_I8 && ragged) {
                    u32x4_t one[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            one[mt][e] = (seen[mt] >> (2 * e) & 1 ? VOP::kOne : 0u) |
                                         (seen[mt] >> (2 * e + 1) & 1 ? VOP::kOne << 16 : 0u);
#pragma unroll
                    for (int c = 0; c < VW; ++c) {
                        uint32_t odd[8], some = 0;
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            odd[r] = not_finite<CODE>(vr[c][r]);
                            some |= odd[r];
                            vr[c][r] &= ~odd[r];
                            odd[r] &= k8 ? 0x38383838u : VOP::kOne | VOP::kOne << 16;     // ones of the type
                        }
                        if (__any(some != 0))
#pragma unroll
                            for (int t = c * (4 / ES); t < (c + 1) * (4 / ES); ++t)
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    const f32x4_t hits = VOP::mfma(column(odd, t), one[mt], (f32x4_t){0, 0, 0, 0});
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        if constexpr (kHitsApart)
                                            hit[mt][t / 8] |= (hits[i] > 0.0f ? 1u : 0u) << (4 * (t % 8) + i);
                                        else
                                            o[mt][t][i] = hits[i] > 0.0f ? nan : o[mt][t][i];
                                }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < CW; ++t) {
                const u32x4_t f = column(vr[t * ES / 4], t);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                    o[mt][t] = VOP::mfma(f, pl[mt], VOP::mfma(f, ph[mt], o[mt][t]));
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v();
        }

        // ---- the waves' parts of the piece: each leaves its rows as they are,
        // and what is read is weighed.  The barriers order LDS only, so that no
        // store to memory is waited for.
        const int ex = opaque(lane), en = ex & 15, eg = ex >> 4, tid = opaque(threadIdx.x);
        const int rows = min(RM, unit.rows - r0);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            if constexpr (kHitsApart)
#pragma unroll
                for (int t = 0; t < CW; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[mt][t][i] = hit[mt][t / 8] >> (4 * (t % 8) + i) & 1 ? nan : o[mt][t][i];
            l[mt] = xor32_sum(xor16_sum(l[mt]));
            // Positions whose scores are all -inf weigh nothing, and are not none: the least
            // finite maximum tells them from a list that names no position.
            if constexpr (MODE == kBlocks)
                m[mt] = named ? fmaxf(m[mt], -__FLT_MAX__) : m[mt];
            if (eg == 0) {
                s_m[wave][16 * mt + en] = m[mt];
                s_l[wave][16 * mt + en] = l[mt];
            }
            if (16 * mt + en < rows)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < CW; t += 4)
                        *(f32x4_t *)&s_o[wave][16 * mt + en][CW * (4 * eg + i) + t] =
                            (f32x4_t){o[mt][t][i], o[mt][t + 1][i], o[mt][t + 2][i], o[mt][t + 3][i]};
        }
        lds_barrier();
        for (int e = tid; e < rows * (DP / 4); e += 64 * kAttWaves) {
            const int r = e / (DP / 4), d = 4 * (e % (DP / 4));
            if (d >= D)
                continue;
            float mx = s_m[0][r], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < kAttWaves; ++w)
                mx = fmaxf(mx, s_m[w][r]);
            const float mu = mx == -INFINITY ? 0.0f : mx;
            f32x4_t y = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kAttWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(s_m[w][r] - mu);
                const f32x4_t v = *(const f32x4_t *)&s_o[w][r][d];
                sum = fmaf(s_l[w][r], f, sum);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    y[i] = fmaf(v[i], f, y[i]);
            }
            if (MODE == kParts || slot >= 0) {
                const int64_t at = (int64_t)slot * a.slot_rows + r;
                *(f32x4_t *)(a.part_o + at * D + d) = y;
                if (d == 0)
                    a.part_ml[at] = make_float2(mx, sum);
                continue;
            }
            const AttendToken t = attend_token(a, unit, r0 + r);
            const int p = s_p[r];
            const float inv = 1.0f / sum;      // no weight at all (every score -inf) gives NaN; zeros where a list names no position
            const float none = MODE == kBlocks && mx == -INFINITY ? 0.0f : nan;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] = p < 0 ? 0.0f : p >= a.cap ? nan : sum == 0.0f ? none : y[i] * inv;
            uint2 w;
            w.x = QOP::pack(y[0], y[1]);
            w.y = QOP::pack(y[2], y[3]);
            *(uint2 *)((char *)a.out + 2 * (((t.b * a.tok.S + t.s) * H * a.G + h * a.G + t.head) * D + d)) = w;
        }
        lds_barrier();
    };

    // ---- a list's segment, cut into equal pieces
    if constexpr (MODE == kBlocks) {
        const uint32_t at = a.first_wg + wg, seg = at / (uint32_t)a.cuts, cut = at - seg * a.cuts;
        const int tiles = (int)(((int64_t)a.take * a.c.page + kAttTile - 1) / kAttTile);
        const uint32_t u = seg / (uint32_t)H;
        piece(u, (int)(seg - u * H), (int)((int64_t)tiles * cut / a.cuts), (int)((int64_t)tiles * (cut + 1) / a.cuts),
              a.cuts > 1 ? (int)at : -1);
        return;
    }

    // ---- one segment a workgroup (workers == 0), or an even share of all tiles
    // in the order unit, cache head, tile.  Every wave counts the units' tiles by
    // itself, 64 units at a time; the host bounds all counts to 32 bits.
    const uint32_t units = a.units;
    auto at_lane = [](uint32_t v, int i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i); };
    const uint32_t segment = a.first_wg + wg;
    uint32_t u = segment / (uint32_t)H;
    int h = (int)(segment - u * H), t0 = -1, t1 = 0, slot = MODE == kParts ? (int)segment : -1;
    uint32_t f = 0, begin = 0, stop = 1, per = 1, total = 0;
    uint32_t first = 0, cost = 0, upto = 0;        // of the lane's unit; of all units up to it in this block of 64
    uint32_t u0 = 0, before = 0;         // the block's first unit; tiles ahead of it
    bool counting = a.workers > 0, load = counting;
    for (;;) {
        if (load) {
            cost = u0 + lane < units ? unit_tiles<RM>(a, u0 + lane, first) + a.piece : 0u;
            upto = cost;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const uint32_t v = __shfl_up(upto, d, 64);
                upto += lane >= d ? v : 0u;
            }
            load = false;
        }
        if (counting) {
            total += at_lane(upto, 63) * H;
            u0 += 64;
            load = u0 < units;
            if (load)
                continue;
            counting = false;
            // At least a tile a wave, and up to two while that leaves a share to
            // every compute unit: one workgroup on each before a second.
            const uint32_t shares = total > 16u * a.few ? a.few : a.workers;
            per = max((total + shares - 1) / shares,
                      min(max((total + 255) / 256, (uint32_t)kAttWaves), 2u * kAttWaves));
            f = begin = min(wg * per, total);
            stop = min(begin + per, total);
            u0 = 0;
            load = units > 64;
            if (load && f < stop)
                continue;
        }
        if (f >= stop)
            return;
        if (a.workers) {
            const uint64_t hit = __ballot(before + upto * H > f);
            if (!hit) {
                before += at_lane(upto, 63) * H;
                u0 += 64;
                load = true;
                if (u0 >= units)           // not reached while positions stay as they are
                    return;
                continue;
            }
            const int i = __builtin_ctzll(hit);
            const uint32_t n1 = at_lane(cost, i), seg0 = before + (at_lane(upto, i) - n1) * H;
            u = u0 + i;
            h = (int)((f - seg0) / n1);
            const uint32_t next = seg0 + (h + 1) * n1, head0 = next - n1 + a.piece;     // the segment's tiles: [head0, next)
            const uint32_t f0 = max(f, head0), f1 = min(next, stop);
            f = f1;
            if (f0 >= f1)
                continue;                  // a share that ends within what a segment's beginning takes
            const int base = (int)at_lane(first, i) - (int)head0;
            t0 = base + (int)f0;
            t1 = base + (int)f1;
            // A piece that begins before its worker's share does is kept in the
            // worker's first slot, else in its second; a whole segment that has
            // to stay a part, in one of its own behind them.
            const bool whole = f0 == head0 && f1 == next;
            slot = 2 * (int)wg + (head0 - a.piece >= begin);
            if (MODE == kParts && whole)
                slot = 2 * a.workers + (int)(u * H) + h;
            if (f0 == head0 && threadIdx.x == 0) {
                const uint32_t w1 = min((next - 1) / per, (uint32_t)a.workers - 1);
                a.desc[u * H + h] = make_int2(slot, (int)(w1 - wg + 1));
            }
            if (MODE == kWhole && whole)
                slot = -1;
        } else
            f = stop;
        piece(u, h, t0, t1, slot);
    }
}

template <typename QOP, int CODE, int KS, int CW, int MT, bool RAGGED>
__global__ void __launch_bounds__(64 * kAttWaves, attend_occupancy(CW, MT, RAGGED && CODE != EP_I8)) attend_kernel(AttendWhole a)
{
    attend_body<QOP, CODE, KS, CW, MT, RAGGED>(a, blockIdx.x);
}
template <typename QOP, int CODE, int KS, int CW, int MT>
__global__ void __launch_bounds__(64 * kAttWaves, attend_occupancy(CW, MT, CODE != EP_I8)) attend_parts_kernel(AttendParts a)
{
    attend_body<QOP, CODE, KS, CW, MT, true>(a, blockIdx.x);
}
template <typename QOP, int CODE, int KS, int CW>
__global__ void __launch_bounds__(64 * kAttWaves, attend_occupancy(CW, 1, false)) attend_blocks_kernel(AttendBlocks a)
{
    attend_body<QOP, CODE, KS, CW, 1, false>(a, blockIdx.x);
}

// Instantiations of one pair of types, by D and rows (attend_gen_*.hip).
template <typename QOP, int CODE, int MT, bool RAGGED>
void attend_by_size(const AttendWhole &a, unsigned grid, hipStream_t st)
{
    constexpr bool k8 = CODE == EP_I8 || CODE == EP_E4M3;
    const int D = a.c.D;
    if (D <= 64)
        attend_kernel<QOP, CODE, 2, 4, MT, RAGGED><<<grid, 64 * kAttWaves, 0, st>>>(a);
    else if (!k8 && D <= 96)
        attend_kernel<QOP, CODE, k8 ? 4 : 3, 8, MT, RAGGED><<<grid, 64 * kAttWaves, 0, st>>>(a);
    else if (D <= 128)
        attend_kernel<QOP, CODE, 4, 8, MT, RAGGED><<<grid, 64 * kAttWaves, 0, st>>>(a);
    else if (D <= 192 && attend_columns(D) == 12)
        attend_kernel<QOP, CODE, 6, 12, MT, RAGGED><<<grid, 64 * kAttWaves, 0, st>>>(a);
    else if (D <= 192)
        attend_kernel<QOP, CODE, 6, 16, MT, RAGGED><<<grid, 64 * kAttWaves, 0, st>>>(a);
    else
        attend_kernel<QOP, CODE, 8, 16, MT, RAGGED><<<grid, 64 * kAttWaves, 0, st>>>(a);
}

template <typename QOP, int CODE>
void attend_by_rows(const AttendWhole &a, int mt, unsigned grid, hipStream_t st)
{
    if (mt == 1 && a.tok.S == 1)
        attend_by_size<QOP, CODE, 1, false>(a, grid, st);
    else if (mt == 1)
        attend_by_size<QOP, CODE, 1, true>(a, grid, st);
    else
        attend_by_size<QOP, CODE, 2, true>(a, grid, st);
}

template <typename QOP, int CODE, int KS, int CW>
void attend_other(const AttendParts &a, int mt, unsigned grid, hipStream_t st)
{
    if (mt == 1)
        attend_parts_kernel<QOP, CODE, KS, CW, 1><<<grid, 64 * kAttWaves, 0, st>>>(a);
    else
        attend_parts_kernel<QOP, CODE, KS, CW, 2><<<grid, 64 * kAttWaves, 0, st>>>(a);
}
template <typename QOP, int CODE, int KS, int CW>
void attend_other(const AttendBlocks &a, int, unsigned grid, hipStream_t st)
{
    attend_blocks_kernel<QOP, CODE, KS, CW><<<grid, 64 * kAttWaves, 0, st>>>(a);
}

// The other kernels, by D (attend_gen_parts.hip, attend_gen_blocks.hip).
template <typename QOP, int CODE, typename ARGS>
void attend_other_by_size(const ARGS &a, int mt, unsigned grid, hipStream_t st)
{
    const int D = a.c.D;
    if (D <= 64)
        attend_other<QOP, CODE, 2, 4>(a, mt, grid, st);
    else if (D <= 128)
        attend_other<QOP, CODE, 4, 8>(a, mt, grid, st);
    else if (D <= 192 && attend_columns(D) == 12)
        attend_other<QOP, CODE, 6, 12>(a, mt, grid, st);
    else if (D <= 192)
        attend_other<QOP, CODE, 6, 16>(a, mt, grid, st);
    else
        attend_other<QOP, CODE, 8, 16>(a, mt, grid, st);
}
template <int CODE, typename ARGS>
void attend_other_by_query(const ARGS &a, int q_dtype, int mt, unsigned grid, hipStream_t st)
{
    if (q_dtype == EP_BF16)
        attend_other_by_size<OpBf16, CODE>(a, mt, grid, st);
    else
        attend_other_by_size<OpF16, CODE>(a, mt, grid, st);
}

void attend_bf16(const AttendWhole &a, int mt, unsigned grid, hipStream_t st);
void attend_f16(const AttendWhole &a, int mt, unsigned grid, hipStream_t st);
void attend_i8(const AttendWhole &a, int q_dtype, int mt, unsigned grid, hipStream_t st);
void attend_e4m3(const AttendWhole &a, int q_dtype, int mt, unsigned grid, hipStream_t st);
// ... and of the other kernels: types from the arguments
void attend_parts(const AttendParts &a, int q_dtype, int mt, unsigned grid, hipStream_t st);
void attend_blocks(const AttendBlocks &a, int q_dtype, unsigned grid, hipStream_t st);

}  // namespace ep
