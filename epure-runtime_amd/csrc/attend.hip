// Attention of new tokens over a paged key-value cache
// (include/epure_paged.h).
//
// One wave per (token, query head): lanes hold the head's values four apart,
// the softmax runs over the positions with a running maximum and sum.
#include "ep_common.h"
#include "ep_internal.h"
#include "ep_paged.h"

namespace ep {
namespace {

struct AttendArgs {
    const void *q;
    int64_t q_sb, q_ss, q_sh;
    int q_dtype, heads;
    PagedTokens tok;
    PagedCache c;
    float scale;
    int64_t window;
    void *out;
    int64_t rows;
};

EP_DEV float cache_value(const PagedCache &c, const void *src, const float *scales, int64_t row, int d)
{
    if (c.dtype == EP_F16 || c.dtype == EP_BF16)
        return load_as_f32(src, c.dtype, row * c.D + d);
    float v[4];
    decode4(((const uint8_t *)src)[row * c.D + d], c.dtype, v);
    return v[0] * scales[row];
}

__global__ void __launch_bounds__(64) attend_kernel(AttendArgs a)
{
    const int lane = threadIdx.x, D = a.c.D;
    const int64_t token = blockIdx.x / a.heads;
    const int h = (int)(blockIdx.x - token * a.heads), kvh = h / (a.heads / a.c.heads);
    const int64_t b = token / a.tok.S, s = token - b * a.tok.S;
    const int64_t p = a.tok.pos[b * a.tok.pos_sb + s * a.tok.pos_ss];
    float q[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
    const int64_t qrow = b * a.q_sb + s * a.q_ss + h * a.q_sh;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        q[i] = lane + 64 * i < D ? load_as_f32(a.q, a.q_dtype, qrow + lane + 64 * i) : 0.0f;
    const int64_t cap = a.tok.width << a.c.page_shift;
    bool bad = p >= cap;
    const int64_t last = p < cap ? p : cap - 1;
    const int64_t first = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    for (int64_t j = first; j <= last; ++j) {
        const int64_t page = a.tok.table[b * a.tok.table_stride + (j >> a.c.page_shift)];
        if (page < 0 || page >= a.c.n_pages) {
            bad = true;
            continue;
        }
        const int64_t row = (page * a.c.heads + kvh) * a.c.page + (j & (a.c.page - 1));
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < D)
                t = fmaf(q[i], cache_value(a.c, a.c.k, a.c.k_scale, row, lane + 64 * i), t);
        t = wave_sum_bfly(t) * a.scale;
        const float n = fmaxf(m, t);
        const float keep = m == -INFINITY ? 0.0f : expf(m - n), w = t == -INFINITY ? 0.0f : expf(t - n);
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < D)
                o[i] = o[i] * keep + w * cache_value(a.c, a.c.v, a.c.v_scale, row, lane + 64 * i);
        m = n;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < D) {
            const float y = bad ? __uint_as_float(0x7fc00000u) : first > last ? 0.0f : o[i] / l;
            store_from_f32(a.out, a.q_dtype, (token * a.heads + h) * D + lane + 64 * i, y);
        }
}

}  // namespace

size_t attend_workspace(const ep_heads *, const PagedTokens &, const PagedCache &) { return 0; }

int launch_attend(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, float scale, int64_t window,
                  void *out, void *, size_t, hipStream_t stream)
{
    AttendArgs a{q->ptr, q->stride_b, q->stride_s, q->stride_h, q->dtype, q->heads, tok, c, scale, window, out,
                 tok.B * tok.S * q->heads};
    if (a.rows == 0)
        return EP_OK;
    if (a.rows > 0x7fffffff)
        return set_error(EP_DECLINE_SHAPE, "%lld rows are more than one launch takes", (long long)a.rows);
    attend_kernel<<<(unsigned)a.rows, 64, 0, stream>>>(a);
    EP_HIP_CHECK(hipGetLastError());
    return EP_OK;
}

}  // namespace ep
