// Descriptors and launchers of the paged-cache kernels (paged.hip,
// attend.hip).  Not part of the public ABI.
#pragma once

#include "ep_common.h"
#include "epure_paged.h"

namespace ep {

struct PagedTokens {
    const int64_t *pos;
    int64_t pos_sb, pos_ss;
    const int32_t *table;
    int64_t table_stride, width;
    int64_t B, S;
};

struct PagedCache {
    void *k, *v;
    float *k_scale, *v_scale;
    int64_t n_pages;
    int dtype, heads, page, page_shift, D;
};

// The values of four 8-bit codes (the scale not applied).
EP_DEV void decode4(uint32_t w, int dtype, float *v)
{
    if (dtype == EP_I8) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = (float)(int8_t)(w >> (8 * i));
    } else {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        v[0] = lo[0];
        v[1] = lo[1];
        v[2] = hi[0];
        v[3] = hi[1];
    }
}

int launch_rotate(const ep_heads *q, const ep_heads *k, const ep_rotation *rot, const PagedTokens &tok, int64_t D,
                  int inverse, void *q_out, void *k_out, hipStream_t stream);
int launch_kv_append(const ep_heads *q, const ep_heads *k, const ep_heads *v, const ep_rotation *rot,
                     const PagedTokens &tok, const PagedCache &c, void *q_out, hipStream_t stream);
int launch_kv_read(const PagedTokens &tok, const PagedCache &c, void *k_out, void *v_out, int out_dtype,
                   hipStream_t stream);
size_t attend_workspace(const ep_heads *q, const PagedTokens &tok, const PagedCache &c);
int launch_attend(const ep_heads *q, const PagedTokens &tok, const PagedCache &c, float scale, int64_t window,
                  void *out, void *ws, size_t ws_bytes, hipStream_t stream);

}  // namespace ep
