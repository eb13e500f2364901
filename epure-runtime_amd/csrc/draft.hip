// Verification of drafted tokens (include/epure_draft.h).
//
//   token x_i stands if u_i q_i(x_i) < p_i(x_i); k of them stand until one does not
//   the next token: the first v with sum_{w <= v} r(w) > u_n sum_w r(w),
//     r = max(p_k - q_k, 0) where a drafted token was turned down, else p_k
//
// in 64 bits, where u q is exact and a sum over the vocabulary is off by some
// 2^-50: the answers are whole numbers and must not hang on the order of sums.
//
// Bound by the bytes of one row of the vocabulary a sequence (of p, and of q
// where a token was turned down): a row is cut into pieces of 1024 values,
// summed side by side; a second launch finds the piece in which the sum is passed
// and looks at it again.  Which tokens stand every workgroup of the first launch
// finds out by itself (a few loads).  64 sequences of 7 drafted tokens over 128256
// (f32, 66 MB of p and q): 13.9 us and 5.2 (8.6 with pieces of 4096); one of 4 over
// 32000: 4.0 and 4.7, a chain of loads and steps over LDS each (5.4 and 7.6).
#include "ep_common.h"
#include "ep_draft.h"
#include "ep_internal.h"

namespace ep {
namespace {

constexpr int kPiece = 1024;

struct DraftArgs {
    DraftTensors t;
    int64_t *accepted, *tokens;
    double2 *part;           // [B][pieces]: sum of r, sum of p
    int64_t *ends;           // [B][2]: drafted tokens that stand; the one turned down, or -1
    uint32_t first_wg, pieces, groups;       // groups: workgroups a sequence of the sums
};

// One probability; a NaN or a negative one is none.
template <typename T>
EP_DEV double prob(const void *p, int64_t at)
{
    const T v = ((const T *)p)[at];
    float f;
    if constexpr (sizeof(T) == 2 && !__is_same(T, f16_t))
        f = bf16_to_f32(v);
    else
        f = (float)v;
    return (double)fmaxf(f, 0.0f);
}

// How many drafted tokens of sequence b stand; turned_down: one that does not
// ended them (-1: the draft ended).  Every wave finds out by itself.
template <typename T>
EP_DEV int stand(const DraftTensors &t, int64_t b, int64_t &turned_down)
{
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < t.n; i0 += 64) {
        const int i = i0 + lane;
        int64_t x = -1;
        bool stands = false;
        if (i < t.n) {
            x = t.drafted[b * t.d_sb + i * t.d_ss];
            x = x < t.V ? x : -1;
            if (x >= 0) {
                const double u = t.uniforms[b * t.u_sb + i * t.u_ss];
                const double q = t.draft ? prob<T>(t.draft, b * t.q_sb + i * t.q_ss + x) : 1.0;
                stands = u * q < prob<T>(t.target, b * t.p_sb + i * t.p_ss + x);
            }
        }
        const uint64_t no = __ballot(!stands);
        if (no && i0 + __builtin_ctzll(no) < t.n) {
            const int l = __builtin_ctzll(no);
            turned_down = __shfl(x, l, 64);
            return i0 + l;
        }
    }
    turned_down = -1;
    return t.n;
}

// r and p of value v.
template <typename T>
EP_DEV double2 weight(const DraftTensors &t, int64_t b, int k, int64_t turned_down, int64_t v)
{
    const double p = prob<T>(t.target, b * t.p_sb + k * t.p_ss + v);
    double q = 0.0;
    if (turned_down >= 0)
        q = t.draft ? prob<T>(t.draft, b * t.q_sb + k * t.q_ss + v) : v == turned_down ? 1.0 : 0.0;
    const double r = p - q;
    return make_double2(r > 0.0 ? r : 0.0, p);
}

EP_DEV double2 wave_sums(double2 v)
{
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) {
        v.x += __shfl_xor(v.x, d, 64);
        v.y += __shfl_xor(v.y, d, 64);
    }
    return v;
}

// A workgroup sums a piece, or (EACH) each of its waves one: what a workgroup
// begins with is then paid for four.
template <typename T, bool EACH>
__global__ void __launch_bounds__(256) sum_kernel(DraftArgs a)
{
    __shared__ double2 s_sum[4];
    const int tid = EACH ? threadIdx.x & 63 : threadIdx.x;
    const uint32_t at = a.first_wg + blockIdx.x, b = at / a.groups, group = at - b * a.groups;
    const uint32_t piece = EACH ? 4 * group + (threadIdx.x >> 6) : group;
    int64_t x;
    const int k = stand<T>(a.t, b, x);
    const int64_t v0 = (int64_t)piece * kPiece;
    const int n = (int)(a.t.V - v0 < kPiece ? a.t.V - v0 : kPiece);
    double2 sum = make_double2(0.0, 0.0);
#pragma unroll 8
    for (int i = tid; i < n; i += EACH ? 64 : 256) {
        const double2 w = weight<T>(a.t, b, k, x, v0 + i);
        sum.x += w.x;
        sum.y += w.y;
    }
    sum = wave_sums(sum);
    if constexpr (!EACH) {
        if ((threadIdx.x & 63) == 0)
            s_sum[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (tid == 0)
            for (int w = 1; w < 4; ++w) {
                sum.x += s_sum[w].x;
                sum.y += s_sum[w].y;
            }
    }
    if (tid == 0 && n > 0) {
        a.part[(int64_t)b * a.pieces + piece] = sum;
        if (piece == 0) {
            a.ends[2 * (int64_t)b] = k;
            a.ends[2 * (int64_t)b + 1] = x;
        }
    }
}

// Sums of the 256 threads' pairs ahead of each thread, and of all.
EP_DEV double2 sums_before(double2 v, double2 *s_wave, double2 &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double2 p = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double x = __shfl_up(p.x, d, 64), y = __shfl_up(p.y, d, 64);
        p.x += lane >= d ? x : 0.0;
        p.y += lane >= d ? y : 0.0;
    }
    const double2 before = make_double2(__shfl_up(p.x, 1, 64), __shfl_up(p.y, 1, 64));
    __syncthreads();
    if (lane == 63)
        s_wave[wave] = p;
    __syncthreads();
    double2 front = make_double2(0.0, 0.0);
    total = front;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w == wave)
            front = total;
        total.x += s_wave[w].x;
        total.y += s_wave[w].y;
    }
    return make_double2(lane ? front.x + before.x : front.x, lane ? front.y + before.y : front.y);
}

// The least `hit` of the threads (none: kNone), else the largest `last`.
constexpr int kNone = 0x7fffffff;
EP_DEV int first_or_last(int hit, int last, int2 *s_wave)
{
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) {
        hit = min(hit, __shfl_xor(hit, d, 64));
        last = max(last, __shfl_xor(last, d, 64));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        s_wave[threadIdx.x >> 6] = make_int2(hit, last);
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
        hit = min(hit, s_wave[w].x);
        last = max(last, s_wave[w].y);
    }
    return hit < kNone ? hit : last;
}

// The piece in which the running sum passes the goal, then the value in it.
// Sums taken in another order may pass it an ulp early or never: what weighs
// nothing is not taken, and where nothing passes, the last that weighs something.
template <typename T>
__global__ void __launch_bounds__(256) pick_kernel(DraftArgs a)
{
    __shared__ double2 s_sums[4];
    __shared__ int2 s_ends[4];
    __shared__ double s_from;
    const uint32_t b = a.first_wg + blockIdx.x;
    const int tid = threadIdx.x;
    const DraftTensors &t = a.t;
    const int k = (int)a.ends[2 * (int64_t)b];
    const int64_t x = a.ends[2 * (int64_t)b + 1];
    const double2 *part = a.part + (int64_t)b * a.pieces;

    // thread i has pieces [i per, (i + 1) per)
    const int per = (int)((a.pieces + 255) / 256), p0 = min(tid * per, (int)a.pieces), p1 = min(p0 + per, (int)a.pieces);
    double2 mine = make_double2(0.0, 0.0), total;
    for (int i = p0; i < p1; ++i) {
        mine.x += part[i].x;
        mine.y += part[i].y;
    }
    double2 run = sums_before(mine, s_sums, total);
    const bool plain = !(total.x > 0.0);         // nothing is left of p - q: p itself
    const double goal = (double)t.uniforms[b * t.u_sb + t.n * t.u_ss] * (plain ? total.y : total.x);
    double at = plain ? run.y : run.x, from = -INFINITY;
    int hit = kNone, last = -1;
    for (int i = p0; i < p1; ++i) {
        const double w = plain ? part[i].y : part[i].x;
        if (!(w > 0.0))
            continue;
        last = i;
        if (hit == kNone && at + w > goal) {
            hit = i;
            from = at;
        }
        at += w;
    }
    const int piece = first_or_last(hit, last, s_ends);
    if (tid == 0)
        s_from = -INFINITY;      // the last piece, and the last value in it
    __syncthreads();
    if (hit == piece)
        s_from = from;
    __syncthreads();
    int64_t v = t.V - 1;         // nothing weighs anything
    if (piece >= 0) {
        constexpr int E = kPiece / 256;          // adjacent values of thread i
        const int64_t v0 = (int64_t)piece * kPiece + tid * E;
        double w[E];
        mine = make_double2(0.0, 0.0);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[e] = 0.0;
            if (v0 + e < t.V) {
                const double2 both = weight<T>(t, b, k, x, v0 + e);
                w[e] = plain ? both.y : both.x;
            }
            mine.x += w[e];
        }
        at = s_from + sums_before(mine, s_sums, total).x;
        hit = kNone;
        last = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            at += w[e];
            if (w[e] > 0.0) {
                last = tid * E + e;
                if (hit == kNone && at > goal)
                    hit = last;
            }
        }
        v = (int64_t)piece * kPiece + first_or_last(hit, last, s_ends);
    }
    int64_t *out = a.tokens + (int64_t)b * (t.n + 1);
    for (int i = tid; i <= t.n; i += 256)
        out[i] = i < k ? t.drafted[b * t.d_sb + i * t.d_ss] : i == k ? v : -1;
    if (tid == 0)
        a.accepted[b] = k;
}

template <typename T>
int launch_typed(DraftArgs a, int64_t B, hipStream_t stream)
{
    // With more pieces than workgroups that the compute units hold at once a wave
    // sums one alone (64 rows of 126 pieces: 21.3 -> 13.7 us; one row of 32: 3.9, 5.4 so).
    const bool each = B * a.pieces > 2048;
    a.groups = each ? (a.pieces + 3) / 4 : a.pieces;
    const int64_t most = 0xffffffff / 256, grid = B * a.groups;
    for (int64_t at = 0; at < grid; at += most) {
        a.first_wg = (uint32_t)at;
        const unsigned n = (unsigned)(grid - at < most ? grid - at : most);
        if (each)
            sum_kernel<T, true><<<n, 256, 0, stream>>>(a);
        else
            sum_kernel<T, false><<<n, 256, 0, stream>>>(a);
        EP_HIP_CHECK(hipGetLastError());
    }
    for (int64_t at = 0; at < B; at += most) {
        a.first_wg = (uint32_t)at;
        pick_kernel<T><<<(unsigned)(B - at < most ? B - at : most), 256, 0, stream>>>(a);
        EP_HIP_CHECK(hipGetLastError());
    }
    return EP_OK;
}

int64_t pieces_of(int64_t V) { return (V + kPiece - 1) / kPiece; }

}  // namespace

size_t verify_workspace(int64_t B, int64_t V) { return (size_t)B * (pieces_of(V) + 1) * sizeof(double2); }

int launch_verify(const DraftTensors &t, int64_t B, int dtype, int64_t *accepted, int64_t *tokens, void *ws,
                  size_t ws_bytes, hipStream_t stream)
{
    const size_t want = verify_workspace(B, t.V);
    if (ws_bytes < want || !ws)
        return set_error(EP_ERR_WORKSPACE, "verification: workspace of %zu bytes, %zu wanted", ws_bytes, want);
    double2 *const part = (double2 *)ws;
    DraftArgs a{t, accepted, tokens, part, (int64_t *)(part + B * pieces_of(t.V)), 0, (uint32_t)pieces_of(t.V), 0};
    if (B > 0x7fffffff / (int64_t)a.pieces)
        return set_error(EP_DECLINE_SHAPE, "%lld sequences over %lld tokens are more than one call takes", (long long)B,
                         (long long)t.V);
    if (dtype == EP_F32)
        return launch_typed<float>(a, B, stream);
    if (dtype == EP_F16)
        return launch_typed<f16_t>(a, B, stream);
    return launch_typed<uint16_t>(a, B, stream);
}

}  // namespace ep
