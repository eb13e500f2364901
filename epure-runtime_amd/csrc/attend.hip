// Attention of new tokens over a paged key-value cache
// (include/epure_paged.h): the plan of a call and the join of its parts.
// The kernel and its layout: attend_kernel.h.
#include <math.h>

#include <algorithm>

#include "attend_kernel.h"

namespace ep {
namespace {

// Joins the pieces of a segment that several workers took, one query row a
// workgroup: D / 4 lanes take a piece, the next ones the next, each with its
// own running maximum, so that sums, maxima and outputs load together.
template <typename OP>
__global__ void __launch_bounds__(256) join_kernel(AttendArgs a, int RM)
{
    __shared__ float s_m[64], s_l[64];
    __shared__ f32x4_t s_y[256];
    const uint32_t Hq = a.c.heads * a.G, D = a.c.D, tid = threadIdx.x;
    const uint32_t out_row = a.first_wg + blockIdx.x, token = out_row / Hq, head = out_row - token * Hq, h = head / a.G, gq = head - h * a.G;
    const uint32_t b = token / (uint32_t)a.tok.S, s = token - b * (uint32_t)a.tok.S;
    const uint32_t row = s * a.G + gq, block = row / RM, r = row - block * RM;
    const int2 d = a.desc[(b * a.blocks + block) * a.c.heads + h];
    const int p = attend_position(a, b, s);
    if (d.y <= 1)       // one worker wrote the output
        return;
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
        for (int k0 = grp; k0 < d.y; k0 += 4 * groups) {
            float2 ml[4];
            f32x4_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // piece 0 is in slot d.x, piece k in the first slot of its worker; past the end the last again
                const int k = min(k0 + i * (int)groups, d.y - 1);
                const int64_t at = (int64_t)(k == 0 ? d.x : (d.x & ~1) + 2 * k) * a.slot_rows + r;
                ml[i] = a.part_ml[at];
                v[i] = *(const f32x4_t *)(a.part_o + at * D + c);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k0 + i * (int)groups < d.y)
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
    for (uint32_t k = 1; k < groups && (int)k < d.y; ++k)
        add(s_m[k], s_l[k], s_y[k * quads + tid]);
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = p < 0 ? 0.0f : p >= a.cap || l == 0.0f ? __uint_as_float(0x7fc00000u) : y[i] * inv;
    uint2 w;
    w.x = OP::pack(y[0], y[1]);
    w.y = OP::pack(y[2], y[3]);
    *(uint2 *)((char *)a.out + 2 * ((int64_t)out_row * D + c)) = w;
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
template <typename F>
int in_launches(int64_t grid, unsigned threads, AttendArgs a, F launch)
{
    const int64_t most = 0xffffffff / threads;
    for (int64_t at = 0; at < grid; at += most) {
        a.first_wg = (uint32_t)at;
        launch(a, (unsigned)std::min(grid - at, most));
        EP_HIP_CHECK(hipGetLastError());
    }
    return EP_OK;
}

}  // namespace

size_t attend_workspace(const ep_heads *q, const PagedTokens &tok, const PagedCache &c)
{
    if (tok.B == 0 || tok.S == 0)
        return 0;
    const Plan p = plan(q, tok, c, 0);
    return p.desc + p.ml + p.o;
}

int launch_attend(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, float scale, int64_t window,
                  void *out, void *ws, size_t ws_bytes, hipStream_t stream)
{
    const Plan p = plan(q, tok, c, window);
    const int64_t cap = tok.width << c.page_shift, rows = tok.S * (q->heads / c.heads), rm = 16 * p.mt;   // cap: below 2^30
    const int64_t out_rows = tok.B * tok.S * q->heads;
    if (rows > 0x3fffffff || p.segments > 0x7fffffff || out_rows > 0x7fffffff)
        return set_error(EP_DECLINE_SHAPE, "%lld query rows are more than one call takes", (long long)out_rows);
    if (ws_bytes < p.desc + p.ml + p.o || (p.workers && !ws))
        return set_error(EP_ERR_WORKSPACE, "attention: workspace of %zu bytes, %zu wanted", ws_bytes,
                         p.desc + p.ml + p.o);
    AttendArgs a{};
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
    a.desc = (int2 *)ws;
    a.part_ml = (float2 *)((char *)ws + p.desc);
    a.part_o = (float *)((char *)ws + p.desc + p.ml);
    const int64_t grid = p.workers ? p.workers : p.segments;
    int rc = in_launches(grid, 64 * kAttWaves, a, [&](const AttendArgs &part, unsigned n) {
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
        // Four groups of lanes where segments are in a few pieces (128 rows x 32
        // heads: 2 us less than eight), eight where one is in hundreds (33 us
        // for 131072 positions on one head, 46 with four).
        const unsigned threads = p.segments * 8 >= p.workers ? 128 : 256;
        rc = in_launches(out_rows, threads, a, [&](const AttendArgs &part, unsigned n) {
            if (q->dtype == EP_BF16)
                join_kernel<OpBf16><<<n, threads, 0, stream>>>(part, (int)rm);
            else
                join_kernel<OpF16><<<n, threads, 0, stream>>>(part, (int)rm);
        });
    }
    return rc;
}

}  // namespace ep
