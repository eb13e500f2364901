// Attention of new tokens over a paged key-value cache
// (include/epure_paged.h): the plan of a call and the join of its parts.
// The kernel and its layout: attend_kernel.h.
#include <math.h>

#include "attend_kernel.h"

namespace ep {
namespace {

// Joins the pieces of a segment that several workers took, one query row a
// workgroup: weights exp2(m_k - max) of the pieces' sums and outputs.
template <typename OP>
__global__ void __launch_bounds__(256) join_kernel(AttendArgs a, int RM)
{
    __shared__ float s_w[256], s_red[8];
    __shared__ f32x4_t s_y[256];
    const int Hq = a.c.heads * a.G, D = a.c.D, tid = threadIdx.x;
    const int64_t token = blockIdx.x / (unsigned)Hq;
    const int head = (int)(blockIdx.x - token * Hq), h = head / a.G, gq = head - h * a.G;
    const int64_t b = token / a.tok.S;
    const int s = (int)(token - b * a.tok.S), row = s * a.G + gq, block = row / RM, r = row - block * RM;
    const int2 d = a.desc[(b * a.blocks + block) * a.c.heads + h];
    if (d.y <= 1)       // one worker wrote the output
        return;
    // piece 0 is in slot d.x, piece k in the first slot of its worker
    auto slot = [&](int k) { return ((int64_t)(k == 0 ? d.x : (d.x & ~1) + 2 * k)) * a.slot_rows + r; };
    auto block_max = [&](float v) {
        v = wave_max(v);
        if ((tid & 63) == 0)
            s_red[tid >> 6] = v;
        __syncthreads();
        v = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        __syncthreads();
        return v;
    };
    float top = -INFINITY;
    for (int k = tid; k < d.y; k += 256)
        top = fmaxf(top, a.part_ml[slot(k)].x);
    top = block_max(top);
    const float base = top == -INFINITY ? 0.0f : top;
    const int quads = D / 4, groups = 256 / quads, grp = tid / quads, c = 4 * (tid - grp * quads);
    f32x4_t y = {0, 0, 0, 0};
    float sum = 0.0f;
    for (int k0 = 0; k0 < d.y; k0 += 256) {
        if (k0 + tid < d.y) {
            const float2 ml = a.part_ml[slot(k0 + tid)];
            s_w[tid] = __builtin_amdgcn_exp2f(ml.x - base);
            sum += ml.y * s_w[tid];
        }
        __syncthreads();
        const int n = min(256, d.y - k0);
        if (grp < groups)
            for (int k = grp; k < n; k += groups) {
                const f32x4_t v = *(const f32x4_t *)(a.part_o + slot(k0 + k) * D + c);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    y[i] = fmaf(v[i], s_w[k], y[i]);
            }
        __syncthreads();
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0)
        s_red[tid >> 6] = sum;
    s_y[tid] = y;
    __syncthreads();
    if (grp != 0)
        return;
    sum = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
    for (int k = 1; k < groups; ++k)
        y += s_y[k * quads + tid];
    const int p = attend_position(a, b, s);
    const float inv = 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = p < 0 ? 0.0f : p >= a.cap || sum == 0.0f ? __uint_as_float(0x7fc00000u) : y[i] * inv;
    uint2 w;
    w.x = OP::pack(y[0], y[1]);
    w.y = OP::pack(y[2], y[3]);
    *(uint2 *)((char *)a.out + 2 * ((token * Hq + head) * D + c)) = w;
}

struct Plan {
    int mt, workers;
    int64_t segments;
    size_t desc, ml, o;     // bytes of the workspace's parts
};

constexpr size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

// Segments of few tiles go to a workgroup each; else all tiles are shared
// evenly among `workers` and the pieces joined.
Plan plan(const ep_heads *q, const PagedTokens &tok, const PagedCache &c)
{
    Plan p{};
    const int64_t rows = tok.S * (q->heads / c.heads);
    p.mt = rows <= 16 ? 1 : 2;
    const int rm = 16 * p.mt;
    p.segments = tok.B * ((rows + rm - 1) / rm) * c.heads;
    const int64_t tiles = (tok.width << c.page_shift) / kAttTile;
    if (tiles > 2 * kAttWaves) {
        p.workers = 256 * 3;
        const size_t slots = (size_t)2 * p.workers * (rows < rm ? rows : rm);
        p.desc = up16(p.segments * sizeof(int2));
        p.ml = up16(slots * sizeof(float2));
        p.o = slots * c.D * sizeof(float);
    }
    return p;
}

}  // namespace

size_t attend_workspace(const ep_heads *q, const PagedTokens &tok, const PagedCache &c)
{
    if (tok.B == 0 || tok.S == 0)
        return 0;
    const Plan p = plan(q, tok, c);
    return p.desc + p.ml + p.o;
}

int launch_attend(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, float scale, int64_t window,
                  void *out, void *ws, size_t ws_bytes, hipStream_t stream)
{
    const Plan p = plan(q, tok, c);
    const int64_t cap = tok.width << c.page_shift, rows = tok.S * (q->heads / c.heads), rm = 16 * p.mt;
    const int64_t out_rows = tok.B * tok.S * q->heads;
    if (cap > 0x3fffffff || rows > 0x3fffffff || p.segments > 0x7fffffff || out_rows > 0x7fffffff)
        return set_error(EP_DECLINE_SHAPE, "%lld positions, %lld query rows: more than one call takes", (long long)cap,
                         (long long)out_rows);
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
    a.units = tok.B * a.blocks;
    a.workers = p.workers;
    a.slot_rows = (int)(rows < rm ? rows : rm);
    a.desc = (int2 *)ws;
    a.part_ml = (float2 *)((char *)ws + p.desc);
    a.part_o = (float *)((char *)ws + p.desc + p.ml);
    const unsigned grid = p.workers ? (unsigned)p.workers : (unsigned)p.segments;
    if (c.dtype == EP_BF16)
        attend_bf16(a, p.mt, grid, stream);
    else if (c.dtype == EP_F16)
        attend_f16(a, p.mt, grid, stream);
    else if (c.dtype == EP_I8)
        attend_i8(a, q->dtype, p.mt, grid, stream);
    else
        attend_e4m3(a, q->dtype, p.mt, grid, stream);
    EP_HIP_CHECK(hipGetLastError());
    if (p.workers) {
        if (q->dtype == EP_BF16)
            join_kernel<OpBf16><<<(unsigned)out_rows, 256, 0, stream>>>(a, (int)rm);
        else
            join_kernel<OpF16><<<(unsigned)out_rows, 256, 0, stream>>>(a, (int)rm);
        EP_HIP_CHECK(hipGetLastError());
    }
    return EP_OK;
}

}  // namespace ep
