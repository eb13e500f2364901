// Attention of new tokens over a paged key-value cache
// (include/epure_paged.h): the plan of a call and the join of its parts.
// The kernel and its layout: attend_kernel.h.
#include <math.h>

#include <algorithm>

#include "attend_front.h"

namespace ep {
namespace {

// Joins `n` pieces of one output row a workgroup, piece k of it at row at(k)
// of the parts: D / 4 lanes take a piece, the next ones the next, each with its
// own running maximum, so that sums, maxima and outputs load together.  p: the
// row's position; none: what a row gives that sees no position (maximum -inf; NaN
// if it has seen some and they weigh nothing).
template <typename OP, typename AT>
EP_DEV void join_row(const AttendArgs &a, int64_t out_row, int p, int n, AT at, float none)
{
    __shared__ float s_m[64], s_l[64];
    __shared__ f32x4_t s_y[256];
    const uint32_t D = a.c.D, tid = threadIdx.x;
    const uint32_t quads = D / 4, groups = blockDim.x / quads, grp = tid / quads, c = 4 * (tid - grp * quads);
    float m = -INFINITY, l = 0.0f;
    f32x4_t y = {0, 0, 0, 0};
    auto add = [&](float m2, float l2, f32x4_t y2) {
        const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
        m = top;
        l = l * f + l2 * f2;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            y[i] = y[i] * f + y2[i] * f2;
    };
    if (grp < groups)
        for (int k0 = grp; k0 < n; k0 += 4 * groups) {
            float2 ml[4];
            f32x4_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t row = at(min(k0 + i * (int)groups, n - 1));      // past the end the last again
                ml[i] = a.part_ml[row];
                v[i] = *(const f32x4_t *)(a.part_o + row * D + c);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k0 + i * (int)groups < n)
                    add(ml[i].x, ml[i].y, v[i]);
        }
    s_y[tid] = y;
    if (grp < groups && c == 0) {
        s_m[grp] = m;
        s_l[grp] = l;
    }
    __syncthreads();
    if (grp != 0)
        return;
    for (uint32_t k = 1; k < groups && (int)k < n; ++k)
        add(s_m[k], s_l[k], s_y[k * quads + tid]);
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = p < 0 ? 0.0f : p >= a.cap ? __uint_as_float(0x7fc00000u) : l == 0.0f ? m == -INFINITY ? none : __uint_as_float(0x7fc00000u) : y[i] * inv;
    uint2 w;
    w.x = OP::pack(y[0], y[1]);
    w.y = OP::pack(y[2], y[3]);
    *(uint2 *)((char *)a.out + 2 * (out_row * D + c)) = w;
}

// An output row: its token (b, s), cache head and place in the group.
struct OutRow {
    uint32_t row, token, b, s, h, gq;
};
EP_DEV OutRow out_row_of(const AttendArgs &a)
{
    const uint32_t Hq = a.c.heads * a.G, row = a.first_wg + blockIdx.x, token = row / Hq, head = row - token * Hq, h = head / a.G;
    const uint32_t b = token / (uint32_t)a.tok.S;
    return {row, token, b, token - b * (uint32_t)a.tok.S, h, head - h * a.G};
}

// Piece k of a segment that several workers took: piece 0 in slot d.x, piece k
// in the first slot of its worker.
EP_DEV int64_t piece_slot(int2 d, int k) { return k == 0 ? d.x : (d.x & ~1) + 2 * k; }

template <typename OP>
__global__ void __launch_bounds__(256) join_kernel(AttendArgs a, int RM)
{
    const OutRow o = out_row_of(a);
    const uint32_t row = o.s * a.G + o.gq, block = row / RM, r = row - block * RM;
    const int2 d = a.desc[(o.b * a.blocks + block) * a.c.heads + o.h];
    const int p = attend_position(a, o.b, o.s);
    if (d.y <= 1)       // one worker wrote the output
        return;
    join_row<OP>(a, o.row, p, d.y, [&](int k) { return piece_slot(d, k) * a.slot_rows + r; }, __uint_as_float(0x7fc00000u));
}

// The pieces over a sequence's own pages, then those over the shared ones.
template <typename OP>
__global__ void __launch_bounds__(256) join_parts_kernel(AttendParts a, int RM)
{
    const OutRow o = out_row_of(a);
    const uint32_t H = a.c.heads;
    const uint32_t row = o.s * a.G + o.gq, block = row / RM, r = row - block * RM;
    const uint32_t all = o.token * a.G + o.gq, rows_f = a.front ? RM : kFrontRows, front = all / rows_f, rf = all - front * rows_f;
    const uint32_t seg = (a.front + o.b * a.blocks + block) * H + o.h, seg_f = front * H + o.h;
    const int2 d = a.workers ? a.desc[seg] : make_int2((int)seg, 1);
    const int2 f = !a.front ? make_int2(0, a.front_splits) : a.workers ? a.desc[seg_f] : make_int2((int)seg_f, 1);
    const int p = attend_position(a, o.b, o.s);
    join_row<OP>(a, o.row, p, d.y + f.y, [&](int k) {
        if (k < d.y)
            return piece_slot(d, k) * a.slot_rows + r;
        k -= d.y;
        return a.front ? piece_slot(f, k) * a.slot_rows + rf : a.front_at + ((int64_t)seg_f * a.front_splits + k) * kFrontRows + rf;
    }, __uint_as_float(0x7fc00000u));
}

template <typename OP>
__global__ void __launch_bounds__(256) join_blocks_kernel(AttendBlocks a)
{
    const OutRow o = out_row_of(a);
    const uint32_t block = o.gq / 16, r = o.gq - 16 * block;
    const int64_t seg = ((int64_t)o.token * a.blocks + block) * a.c.heads + o.h;
    const int p = attend_position(a, o.b, o.s);
    join_row<OP>(a, o.row, p, a.cuts, [&](int k) { return (seg * a.cuts + k) * a.slot_rows + r; }, 0.0f);
}

struct Plan {
    int mt, workers;
    int64_t segments;
    size_t desc, ml, o;     // bytes of the workspace's parts
};

int row_bytes(const PagedCache &c) { return c.D * (c.dtype == EP_F16 || c.dtype == EP_BF16 ? 2 : 1); }

// A piece takes some 6 us beyond its tiles, and a tile as long as a worker's
// part of the bandwidth needs for its bytes: 6 tiles' time for 128 16-bit
// values and 512 workers.  Short sequences of a ragged batch cost that much
// more than their lengths say (a worker that got a dozen of them took 97 us
// where the rest took 46).
constexpr int kMostPiece = 786432 / (16 * 256);
int piece_tiles(const PagedCache &c, int workers)
{
    return 786432 / (row_bytes(c) * std::max(workers, 256));
}

constexpr size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

// Segments of few tiles go to a workgroup each: up to 16 tiles, or up to 32
// the more segments there are to fill the compute units (8 segments of 22 tiles
// take 11.4 us so, 10.2 shared; 64 of 19, 12.0 and 13.1; 128 of 19, 12.5 and
// 17.2; 512 of 16, 17 and 22; 256 of 1 to 128, 64 and 59).  Else all tiles are
// shared evenly among `workers`, as many workgroups as are resident at once,
// and the pieces joined (where 32 bits count all tiles that the table could
// hold).
//
// A long call goes to one workgroup a compute unit where its four waves' tiles
// are 12 KiB each: what is in flight is enough, and there are half as many
// pieces (4 x 131072 bf16 positions of 128 values 301 us, 307 with two; one
// head of 131072 27 and 33; 32 rows a key head 48 and 51; 192 int8 values, 4 x
// 131072 positions 280 and 283, one head 31 and 41, 16 x 2-8 thousand 34.4 and
// 33.3).  Smaller tiles need the second one (48 x 8192 in int8: 107 us with
// one, 86 with two; of 80 bf16 values 31.5 and 29.3), and short calls both (one
// sequence of 8000: 15.9 and 15.2).
Plan plan(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, int64_t window)
{
    Plan p{};
    const int64_t rows = tok.S * (q->heads / c.heads);
    p.mt = rows <= 16 ? 1 : 2;
    const int rm = 16 * p.mt;
    p.segments = tok.B * ((rows + rm - 1) / rm) * c.heads;
    const int64_t tiles = (tok.width << c.page_shift) / kAttTile;
    // a window's tiles, if the call's tokens follow one another
    const int64_t most = window > 0 && window <= tiles * kAttTile
                             ? std::min(tiles, (window + tok.S) / kAttTile + 2) : tiles;
    if (most > std::min<int64_t>(16 + p.segments / 8, 32) && p.segments < 0x40000000 && tiles + kMostPiece < 0x7fff0000 / p.segments) {
        p.workers = 256 * attend_occupancy(attend_columns(c.D), p.mt, tok.S > 1 && c.dtype != EP_I8);
        const size_t slots = (size_t)2 * p.workers * (rows < rm ? rows : rm);
        p.desc = up16(p.segments * sizeof(int2));
        p.ml = up16(slots * sizeof(float2));
        p.o = slots * c.D * sizeof(float);
    }
    return p;
}

// A launch has fewer than 2^32 threads: a grid beyond that is cut into several.
template <typename ARGS, typename F>
int in_launches(int64_t grid, unsigned threads, ARGS a, F launch)
{
    const int64_t most = 0xffffffff / threads;
    for (int64_t at = 0; at < grid; at += most) {
        a.first_wg = (uint32_t)at;
        launch(a, (unsigned)std::min(grid - at, most));
        EP_HIP_CHECK(hipGetLastError());
    }
    return EP_OK;
}

// Four groups of lanes where segments are in a few pieces (128 rows x 32
// heads: 2 us less than eight), eight where one is in hundreds (33 us for
// 131072 positions on one head, 46 with four).
unsigned join_threads(int64_t segments, int workers) { return segments * 8 >= workers ? 128 : 256; }

// What every call's kernels are given.
void fill(AttendArgs &a, const ep_heads *q, const PagedTokens &tok, const PagedCache &c, float scale, int64_t window,
          void *out)
{
    const int64_t cap = tok.width << c.page_shift;      // below 2^30
    a.q = q->ptr;
    a.q_sb = q->stride_b;
    a.q_ss = q->stride_s;
    a.q_sh = q->stride_h;
    a.tok = tok;
    a.c = c;
    a.scale = scale * (float)M_LOG2E;
    a.cap = (int)cap;
    a.window = window > 0 && window < cap ? (int)window : (int)cap;
    a.out = out;
    a.G = q->heads / c.heads;
}

// The workspace's parts: descriptors, maxima and sums, outputs.
template <typename PLAN>
int give(AttendArgs &a, const PLAN &p, void *ws, size_t ws_bytes)
{
    if (ws_bytes < p.desc + p.ml + p.o || (p.desc + p.ml + p.o && !ws))
        return set_error(EP_ERR_WORKSPACE, "attention: workspace of %zu bytes, %zu wanted", ws_bytes,
                         p.desc + p.ml + p.o);
    a.desc = (int2 *)ws;
    a.part_ml = (float2 *)((char *)ws + p.desc);
    a.part_o = (float *)((char *)ws + p.desc + p.ml);
    return EP_OK;
}

bool too_many_rows(int64_t rows, int64_t segments, int64_t out_rows)
{
    return rows > 0x3fffffff || segments > 0x7fffffff || out_rows > 0x7fffffff;
}

struct PartsPlan {
    int mt, workers;
    int64_t blocks, front, segments;
    size_t desc, ml, o;
    int slot_rows;
    int64_t groups, splits, slots;       // of attend_front.h (groups 0: not used); slots of the others
};

// Pieces that the shared positions are cut into for `groups` row groups of all
// cache heads: the fewest that fill the room for workgroups, round by round (else
// those that fill it best), of four stages at least, as every row of every piece is
// written and joined (32 x 4 rows on 8 heads over 8192 positions: 32 pieces of
// four 26.8 us, 64 of two 33.7), or of two up to 128 workgroups (16 x 4 over 2048:
// 8 pieces of four 18.4 us, 16 of two 15.7).
int64_t front_splits(int64_t groups, int64_t stages)
{
    const int64_t room = 256 * kFrontOccupancy;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(std::max(stages / 4, std::min(stages / 2, (127 + groups) / groups)), 256));
    int64_t best = 1;
    double best_full = 0.0;
    for (int64_t s = 1; s <= most; ++s) {
        const int64_t n = groups * s;
        const double full = (double)n / (double)(room * ((n + room - 1) / room));
        if (full > best_full) {
            best = s;
            best_full = full;
        }
        if (full >= 0.97)
            break;
    }
    return best;
}

// Whether the shared pages go through LDS (attend_front.h): from 33 rows a cache
// head on, if those of one sequence are a tile at most (16 x 4 rows on 8 heads over
// 1024 positions 18.0 us as units, 14.0 so; 32 x 4 over 8192 37.8 and 28.2; 64 x 4
// over 65536 351 and 157 to 164; 2 x 4 over 8192, where most of a workgroup's rows are none,
// 18.3 and 19.9), or from 16384 tiles of 32 rows by 32 positions on (16 x 32 rows on
// 8 heads over 4096, 16384 tiles, 45.6 and 38.8; 9 x 25 on 4 of 80 over 2992, 2992
// tiles, 21.5 and 22.8, of e4m3 with a window 22.0 and 26.6).
// Where a window may end among the shared pages, scores there are masked one by
// one, and 256 rows are asked for (window 40 short of the pages, as units and so:
// 16 x 4 over 4096 22.6 and 32.5, of e4m3 22.0 and 35.7; 64 x 4 over 2048 36.2 and
// 35.8, of e4m3 37.1 and 38.9; windows of 1100: 20.1 and 17.0, 32.9 and 25.8; what
// lies between 64 and 256 rows was not measured).  The host knows no positions: a
// window shorter than the table counts, though it may be longer than any context.
// Up to 32 rows of one sequence go in the same launch as those pages do; more go in
// one of their own behind it, which takes 32 at a time.
constexpr int kTogetherRows = 32;
constexpr int64_t kTogether = 0x800000;      // workgroups of one launch of both kinds
bool through_lds(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, int64_t shared, int64_t window)
{
    const int64_t rows = tok.S * (q->heads / c.heads), all = tok.B * rows;
    int64_t seen = shared << c.page_shift;
    if (window > 0)
        seen = std::min(seen, window);
    const bool cut = window > 0 && window < tok.width << c.page_shift;
    return all > 32 && c.D <= kFrontWidest &&
           ((rows <= 16 && (!cut || all >= 256)) || (all + 31) / 32 * c.heads >= 16384 / std::max<int64_t>(seen / kAttTile, 1));
}

// Units of the whole batch over the shared pages, then the sequences' own:
// as plan() does, but that every segment leaves a part.  dense: the former go
// through LDS instead.
PartsPlan plan_parts(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, int64_t shared, int64_t window, bool dense)
{
    PartsPlan p{};
    const int64_t rows = tok.S * (q->heads / c.heads), all = tok.B * rows;
    p.mt = (dense ? rows <= kTogetherRows : all <= 16) ? 1 : 2;
    const int64_t rm = 16 * p.mt;
    p.blocks = (rows + rm - 1) / rm;
    p.front = dense ? 0 : (all + rm - 1) / rm;
    p.segments = (p.front + tok.B * p.blocks) * c.heads;
    p.slot_rows = (int)std::min(dense ? rows : all, rm);
    if (dense) {
        p.groups = (all + kFrontRows - 1) / kFrontRows;
        p.splits = front_splits(p.groups * c.heads, ((shared << c.page_shift) + kFrontStage - 1) / kFrontStage);
    }
    const int64_t tiles = ((dense ? tok.width - shared : std::max(shared, tok.width - shared)) << c.page_shift) / kAttTile + 1;
    const int64_t most = window > 0 && window <= tiles * kAttTile
                             ? std::min(tiles, (window + tok.S) / kAttTile + 2) : tiles;
    if (most > std::min<int64_t>(16 + p.segments / 8, 32) && p.segments < 0x40000000 && tiles + kMostPiece < 0x7fff0000 / p.segments)
        p.workers = 256 * (dense && p.mt == 1 ? 1 : attend_occupancy(attend_columns(c.D), p.mt, c.dtype != EP_I8));
    p.slots = ((int64_t)2 * p.workers + p.segments) * p.slot_rows;
    const size_t part_rows = (size_t)p.slots + (size_t)p.groups * c.heads * p.splits * kFrontRows;
    p.desc = p.workers ? up16(p.segments * sizeof(int2)) : 0;
    p.ml = up16(part_rows * sizeof(float2));
    p.o = part_rows * c.D * sizeof(float);
    return p;
}

struct BlocksPlan {
    int64_t blocks, segments;
    int cuts, slot_rows;
    size_t desc, ml, o;
};

// A list of few tiles goes to a workgroup as a whole (as in plan(): 16, or up
// to 32 the more lists there are); else it is cut into as many pieces as fill the
// compute units twice, of eight tiles at least (two a wave).
BlocksPlan plan_blocks(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, int64_t take)
{
    BlocksPlan p{};
    const int64_t G = q->heads / c.heads, tiles = (take * c.page + kAttTile - 1) / kAttTile;
    p.blocks = (G + 15) / 16;
    p.segments = tok.B * tok.S * p.blocks * c.heads;
    p.cuts = 1;
    if (tiles > std::min<int64_t>(16 + p.segments / 8, 32))
        p.cuts = (int)std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(p.segments, 1), tiles / (2 * kAttWaves)));
    p.slot_rows = (int)std::min<int64_t>(G, 16);
    if (p.cuts > 1) {
        const size_t slots = (size_t)p.segments * p.cuts * p.slot_rows;
        p.ml = up16(slots * sizeof(float2));
        p.o = slots * c.D * sizeof(float);
    }
    return p;
}

// Sharing pays where there is more than one sequence, and from 1024 positions
// seen on (16 x 4 rows on 8 heads behind 512 and 1024: 12.0 and 19.6 us each for
// itself, 14.0 and 14.3 shared; 64 x 4 behind 1024: 36 and 22; 32 x 4 with 1024 of
// their own behind 512 and 2048: 31.7 and 46, 31.8 and 34).
bool shares(const PagedTokens &tok, const PagedCache &c, int64_t shared, int64_t window)
{
    return tok.B > 1 && shared << c.page_shift >= 1024 && (window <= 0 || window >= 1024);
}

}  // namespace

size_t attend_workspace(const ep_heads *q, const PagedTokens &tok, const PagedCache &c)
{
    if (tok.B == 0 || tok.S == 0)
        return 0;
    const Plan p = plan(q, tok, c, 0);
    return p.desc + p.ml + p.o;
}

size_t attend_parts_workspace(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, int64_t shared)
{
    if (tok.B == 0 || tok.S == 0)
        return 0;
    // a window may turn the choices
    size_t most = attend_workspace(q, tok, c);
    if (!shares(tok, c, shared, 0))
        return most;
    for (const bool dense : {false, through_lds(q, tok, c, shared, 0)}) {
        const PartsPlan p = plan_parts(q, tok, c, shared, 0, dense);
        most = std::max(most, p.desc + p.ml + p.o);
    }
    return most;
}

size_t attend_blocks_workspace(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, int64_t take)
{
    if (tok.B == 0 || tok.S == 0 || take == 0)
        return 0;
    const BlocksPlan p = plan_blocks(q, tok, c, take);
    return p.ml + p.o;
}

int launch_attend(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, float scale, int64_t window,
                  void *out, void *ws, size_t ws_bytes, hipStream_t stream)
{
    const Plan p = plan(q, tok, c, window);
    const int64_t rows = tok.S * (q->heads / c.heads), rm = 16 * p.mt;
    const int64_t out_rows = tok.B * tok.S * q->heads;
    if (too_many_rows(rows, p.segments, out_rows))
        return set_error(EP_DECLINE_SHAPE, "%lld query rows are more than one call takes", (long long)out_rows);
    AttendWhole a{};
    int rc = give(a, p, ws, ws_bytes);
    if (rc != EP_OK)
        return rc;
    fill(a, q, tok, c, scale, window, out);
    a.rows = (int)rows;
    a.blocks = (int)((rows + rm - 1) / rm);
    a.units = (uint32_t)(tok.B * a.blocks);
    a.workers = p.workers;
    a.few = row_bytes(c) >= 192 ? 256 : p.workers;
    a.piece = piece_tiles(c, p.workers);
    // Values pass the caches on their way (4 x 131072 positions in 313 us, 348
    // with plain loads).  Keys do too (308) unless they are read again soon: by
    // a sequence's next unit in this call (64 rows a key head: 85 us, 79 with
    // plain key loads), or by the next call where the 256 MB behind the L2
    // caches hold a few such pools (16 x 2-4 thousand int8 positions: 28.7, 26.9).
    a.keys_once = a.blocks == 1 && c.n_pages * c.heads * c.page * row_bytes(c) > (int64_t)80 << 20;
    a.slot_rows = (int)(rows < rm ? rows : rm);
    const int64_t grid = p.workers ? p.workers : p.segments;
    rc = in_launches(grid, 64 * kAttWaves, a, [&](const AttendWhole &part, unsigned n) {
        if (c.dtype == EP_BF16)
            attend_bf16(part, p.mt, n, stream);
        else if (c.dtype == EP_F16)
            attend_f16(part, p.mt, n, stream);
        else if (c.dtype == EP_I8)
            attend_i8(part, q->dtype, p.mt, n, stream);
        else
            attend_e4m3(part, q->dtype, p.mt, n, stream);
    });
    if (rc == EP_OK && p.workers) {
        const unsigned threads = join_threads(p.segments, p.workers);
        rc = in_launches(out_rows, threads, a, [&](const AttendWhole &part, unsigned n) {
            if (q->dtype == EP_BF16)
                join_kernel<OpBf16><<<n, threads, 0, stream>>>(part, (int)rm);
            else
                join_kernel<OpF16><<<n, threads, 0, stream>>>(part, (int)rm);
        });
    }
    return rc;
}

int launch_attend_parts(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, int64_t shared, float scale,
                        int64_t window, void *out, void *ws, size_t ws_bytes, hipStream_t stream)
{
    if (!shares(tok, c, shared, window))
        return launch_attend(q, tok, c, scale, window, out, ws, ws_bytes, stream);
    const PartsPlan p = plan_parts(q, tok, c, shared, window, through_lds(q, tok, c, shared, window));
    const int64_t rows = tok.S * (q->heads / c.heads), rm = 16 * p.mt;
    const int64_t out_rows = tok.B * tok.S * q->heads;
    if (too_many_rows(tok.B * rows, p.segments + 2 * p.workers, out_rows))
        return set_error(EP_DECLINE_SHAPE, "%lld query rows are more than one call takes", (long long)out_rows);
    AttendParts a{};
    int rc = give(a, p, ws, ws_bytes);
    if (rc != EP_OK)
        return rc;
    fill(a, q, tok, c, scale, window, out);
    a.rows = (int)rows;
    a.blocks = (int)p.blocks;
    a.front = (int)p.front;
    a.front_rows = (int)(tok.B * rows);
    a.shared = (int)shared;
    a.from = (int)(shared << c.page_shift);
    a.units = (uint32_t)(p.front + tok.B * p.blocks);
    a.workers = p.workers;
    a.few = p.workers;
    a.piece = piece_tiles(c, p.workers);
    a.slot_rows = p.slot_rows;
    a.front_splits = (int)p.splits;
    a.front_at = p.slots;
    const int64_t grid = p.workers ? p.workers : p.segments;
    bool apart = true;
    if (p.groups) {
        FrontArgs f{};
        f.q = a.q;
        f.q_sb = a.q_sb;
        f.q_ss = a.q_ss;
        f.q_sh = a.q_sh;
        f.tok = tok;
        f.c = c;
        f.scale = a.scale;
        f.window = a.window;
        f.cap = a.cap;
        f.G = a.G;
        f.rows = a.front_rows;
        f.limit = a.from;
        f.groups = (int)p.groups;
        f.splits = (int)p.splits;
        f.part_ml = a.part_ml + p.slots;
        f.part_o = a.part_o + p.slots * c.D;
        const int64_t pairs = (int64_t)c.heads * p.splits, fronts = (pairs + 7) / 8 * 8 * p.groups;
        if (p.mt == 1 && fronts + grid <= kTogether) {
            attend_front_tails(FrontTails{f, a, (uint32_t)fronts}, q->dtype, (unsigned)(fronts + grid), stream);
            EP_HIP_CHECK(hipGetLastError());
            apart = false;
        } else
            rc = in_launches(fronts, 64 * kFrontWaves, f,
                             [&](const FrontArgs &part, unsigned n) { attend_front(part, q->dtype, n, stream); });
        if (rc != EP_OK)
            return rc;
    }
    if (apart)
        rc = in_launches(grid, 64 * kAttWaves, a, [&](const AttendParts &part, unsigned n) {
            attend_parts(part, q->dtype, p.mt, n, stream);
        });
    if (rc == EP_OK) {
        const unsigned threads = join_threads(p.segments, p.workers);
        rc = in_launches(out_rows, threads, a, [&](const AttendParts &part, unsigned n) {
            if (q->dtype == EP_BF16)
                join_parts_kernel<OpBf16><<<n, threads, 0, stream>>>(part, (int)rm);
            else
                join_parts_kernel<OpF16><<<n, threads, 0, stream>>>(part, (int)rm);
        });
    }
    return rc;
}

int launch_attend_blocks(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, const int32_t *list,
                         int64_t take, float scale, int64_t window, void *out, void *ws, size_t ws_bytes,
                         hipStream_t stream)
{
    const BlocksPlan p = plan_blocks(q, tok, c, take);
    const int64_t out_rows = tok.B * tok.S * q->heads;
    if (take > (0x3fffffff >> c.page_shift) || p.segments * p.cuts > 0x7fffffff || out_rows > 0x7fffffff)
        return set_error(EP_DECLINE_SHAPE, "%lld query rows over %lld pages each are more than one call takes",
                         (long long)out_rows, (long long)take);
    AttendBlocks a{};
    int rc = give(a, p, ws, ws_bytes);
    if (rc != EP_OK)
        return rc;
    fill(a, q, tok, c, scale, window, out);
    a.blocks = (int)p.blocks;
    a.list = list;
    a.take = (int)take;
    a.cuts = p.cuts;
    a.slot_rows = p.slot_rows;
    rc = in_launches(p.segments * p.cuts, 64 * kAttWaves, a, [&](const AttendBlocks &part, unsigned n) {
        attend_blocks(part, q->dtype, n, stream);
    });
    if (rc == EP_OK && p.cuts > 1)
        rc = in_launches(out_rows, 128, a, [&](const AttendBlocks &part, unsigned n) {
            if (q->dtype == EP_BF16)
                join_blocks_kernel<OpBf16><<<n, 128, 0, stream>>>(part);
            else
                join_blocks_kernel<OpF16><<<n, 128, 0, stream>>>(part);
        });
    return rc;
}

}  // namespace ep
