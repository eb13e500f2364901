// Rotary positions, and the rows of a paged key-value cache: written (turned
// and quantised on the way) and read back.  Declared in
// include/epure_paged.h; attention over the cache is attend.hip.
//
// One kernel shape serves all three: a row is one head's D values of one
// token, a lane holds 16 of them as two 16-byte chunks, and D / 16 lanes
// (rounded up to a power of two) hold a row.  The chunks lie dim / 2 apart
// (D / 2 without a turn): with pairs (i, i + dim / 2) a turn needs nothing
// from another lane, in either layout neighbouring lanes load and store
// neighbouring chunks, and a row's largest magnitude is a few lane exchanges
// within 16 lanes.
//
// All of it is bound by the bytes of the rows.  Inputs are read once, and
// large outputs leave the caches before they are read again, so both go past
// them as non-temporal accesses: 16384 tokens of 32 + 8 heads of 128 turn in
// 58 us (5.8 TB/s; 70 with plain accesses), 8 x 4096 rows of 8 heads are read
// out of an int8 cache in 35 us (50), two prompts of 4096 tokens enter an
// e4m3 cache and are read back in 46 us (60).  Four rows of one token a group
// of lanes, with one look-up of position, page and angles, were slower: lanes
// of a wave then hold queries, keys and values at once and take every path
// (those prompts 124 us), and one token's call grows with the code it fetches.
// Position and row load side by side, page and angles after them: with the row
// behind the position those prompts took 49.5 us, 8 tokens 3.4 instead of 3.2.
#include "ep_common.h"
#include "ep_internal.h"
#include "ep_paged.h"

namespace ep {
namespace {

struct Turn {
    const float *cos_t, *sin_t;
    int64_t max_pos;
    int dim;          // 0: no rotation
    int interleaved;
    float sign;       // -1: the inverse
};

struct Rows {
    const void *ptr;
    int64_t sb, ss, sh;
    int heads;
};

// a or b, field by field: a choice between two of the kernel's arguments by
// address would load them from memory once more.
EP_DEV Rows pick(bool first, const Rows &a, const Rows &b)
{
    return {first ? a.ptr : b.ptr, first ? a.sb : b.sb, first ? a.ss : b.ss, first ? a.sh : b.sh,
            first ? a.heads : b.heads};
}

// Element index (within its row) of value e of a lane: chunk a, then chunk b.
struct Chunks {
    int a, b;
    EP_DEV int at(int e) const { return e < 8 ? a + e : b + e - 8; }
};

// Lane u's chunks where whole chunks can be loaded: half of the turned values
// apart (dim 0: no turn), or half of the others.
EP_DEV Chunks chunks_of(int u, int dim, int D)
{
    const int w = u - dim / 16;
    return w < 0 ? Chunks{8 * u, 8 * u + dim / 2} : Chunks{dim + 8 * w, dim + 8 * w + (D - dim) / 2};
}

template <typename T>
EP_DEV float to_f32(T v);
template <>
EP_DEV float to_f32<float>(float v) { return v; }
template <>
EP_DEV float to_f32<f16_t>(f16_t v) { return (float)v; }
template <>
EP_DEV float to_f32<uint16_t>(uint16_t v) { return bf16_to_f32(v); }

template <typename T>
EP_DEV T from_f32(float v);
template <>
EP_DEV float from_f32<float>(float v) { return v; }
template <>
EP_DEV f16_t from_f32<f16_t>(float v) { return (f16_t)v; }
template <>
EP_DEV uint16_t from_f32<uint16_t>(float v) { return f32_to_bf16(v); }

// 8 values in 16-byte aligned memory, as they lie there.  Loads of what is
// read once.
template <typename T>
struct Raw8 {
    u32x4_t w[sizeof(T) / 2];
    EP_DEV void load(const T *p)
    {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i)
            w[i] = __builtin_nontemporal_load((const u32x4_t *)p + i);
    }
    EP_DEV void widen(float *v) const
    {
        T r[8];
        __builtin_memcpy(r, w, sizeof r);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = to_f32<T>(r[i]);
    }
};

template <typename T>
EP_DEV void load8(const T *p, float *v)
{
    Raw8<T> r;
    r.load(p);
    r.widen(v);
}
// STREAM: past the caches (a parameter of the kernels: a branch's two stores
// would be merged into one plain store).
template <bool STREAM, typename T>
EP_DEV void store8(T *p, const float *v)
{
    T r[8];
    u32x4_t w[sizeof r / 16];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        r[i] = from_f32<T>(v[i]);
    __builtin_memcpy(w, r, sizeof r);
#pragma unroll
    for (unsigned i = 0; i < sizeof r / 16; ++i)
        if constexpr (STREAM)
            __builtin_nontemporal_store(w[i], (u32x4_t *)p + i);
        else
            ((u32x4_t *)p)[i] = w[i];
}

// (a cos - b sin, b cos + a sin), each product rounded before the sum: the
// result is the one of elementary f32 operations, whatever the compiler
// would contract (an 8-bit code next to a rounding border depends on it).
EP_DEV void turn_pair(float a, float b, float c, float s, float &ta, float &tb)
{
#pragma clang fp contract(off)
    const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
    ta = ac - bs;
    tb = bc + as;
}

// The 16 values of lane u of the row at x.  VEC: chunks are loaded whole (D
// and, with a turn, dim / 2 in whole chunks, everything 16-byte aligned); else
// value by value (16384 tokens of 40 heads of 80 values: 254 us with 40 of them
// turned, 57 with all).  load() needs no position and goes ahead of what waits for
// one; values() then turns by position p (in the tables) where `turned`.
template <typename T, bool VEC>
struct LaneRow {
    const T *x;
    int D, u;
    Chunks ch;
    Raw8<T> a, b;

    EP_DEV void load(const T *src, int D_, int u_, const Turn &t)
    {
        x = src;
        D = D_;
        u = u_;
        ch = VEC ? chunks_of(u, t.dim, D) : Chunks{16 * u, 16 * u + 8};
        if constexpr (VEC) {
            a.load(x + ch.a);
            b.load(x + ch.b);
        }
    }
    EP_DEV void values(const Turn &t, bool turned, int64_t p, float *v) const
    {
        const int half = t.dim / 2;
        if constexpr (VEC) {
            // cosines and sines of the pairs of both chunks (of some row, not
            // used, where nothing turns: a branch would part the loads)
            float c[8], s[8];
            const bool turns = turned && 16 * u < t.dim;
            if (t.max_pos > 0) {
                const int64_t at = turns ? p * half + (t.interleaved ? ch.a / 2 : ch.a) : 0;
                const int64_t next = turns ? p * half + (t.interleaved ? ch.b / 2 : ch.a + 4) : 0;
                __builtin_memcpy(c, __builtin_assume_aligned(t.cos_t + at, 16), 16);
                __builtin_memcpy(c + 4, __builtin_assume_aligned(t.cos_t + next, 16), 16);
                __builtin_memcpy(s, __builtin_assume_aligned(t.sin_t + at, 16), 16);
                __builtin_memcpy(s + 4, __builtin_assume_aligned(t.sin_t + next, 16), 16);
            }
            a.widen(v);
            b.widen(v + 8);
            if (!turns)
                return;
            if (t.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    turn_pair(v[2 * i], v[2 * i + 1], c[i], t.sign * s[i], v[2 * i], v[2 * i + 1]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    turn_pair(v[i], v[i + 8], c[i], t.sign * s[i], v[i], v[i + 8]);
            }
        } else {
            for (int e = 0; e < 16; ++e) {
                const int d = 16 * u + e;
                v[e] = d < D ? to_f32<T>(x[d]) : 0.0f;
                if (turned && d < t.dim) {
                    const bool second = t.interleaved ? (d & 1) : d >= half;
                    const int i = t.interleaved ? d >> 1 : (second ? d - half : d);
                    const int other = t.interleaved ? d ^ 1 : (second ? d - half : d + half);
                    const float y = to_f32<T>(x[other]), c = t.cos_t[p * half + i], s = t.sign * t.sin_t[p * half + i];
                    float ta, tb;
                    if (second)
                        turn_pair(y, v[e], c, s, ta, tb);
                    else
                        turn_pair(v[e], y, c, s, ta, tb);
                    v[e] = second ? tb : ta;
                }
            }
        }
    }
};

template <bool VEC, bool STREAM, typename T>
EP_DEV void store_row(T *y, int D, const Chunks &ch, const float *v)
{
    if constexpr (VEC) {
        store8<STREAM>(y + ch.a, v);
        store8<STREAM>(y + ch.b, v + 8);
    } else {
        for (int e = 0; e < 16; ++e)
            if (ch.at(e) < D)
                y[ch.at(e)] = from_f32<T>(v[e]);
    }
}

// Largest over the lanes (a power of two, at most 16) that hold a row:
// quads, then lane mirrors within 8 and 16 (every lane of the row takes
// part; lanes of one row are adjacent and aligned).
EP_DEV uint32_t row_max(uint32_t m, int lanes)
{
    auto step = [&](uint32_t o) { m = m > o ? m : o; };
    if (lanes > 1)
        step(__builtin_amdgcn_update_dpp(0, m, 0xb1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
    if (lanes > 2)
        step(__builtin_amdgcn_update_dpp(0, m, 0x4e, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
    if (lanes > 4)
        step(__builtin_amdgcn_update_dpp(0, m, 0x141, 0xf, 0xf, false));  // row_half_mirror
    if (lanes > 8)
        step(__builtin_amdgcn_update_dpp(0, m, 0x140, 0xf, 0xf, false));  // row_mirror
    return m;
}

EP_DEV float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Scale and codes of a lane's 16 values of a row whose largest |x| has the
// bits `m` (as integers, magnitudes order NaN above infinity above the rest).
EP_DEV float quantise(const float *v, uint32_t m, int dtype, uint32_t *codes)
{
    if (m >= 0x7f800000u) {
        codes[0] = codes[1] = codes[2] = codes[3] = 0;
        return __uint_as_float(0x7fc00000u);
    }
    if (dtype == EP_I8) {
        const float top = fmaxf(__uint_as_float(m), pow2(-100));
        const float inv = 127.0f / top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float q = fminf(fmaxf(rintf(v[4 * i + j] * inv), -127.0f), 127.0f);
                w |= ((uint32_t)(int)q & 0xffu) << (8 * j);
            }
            codes[i] = w;
        }
        return top / 127.0f;
    }
    // 448 = 0.875 * 2^9: m = f * 2^n with f in [0.5, 1) fits 448 * 2^e from
    // e = n - 9 where f <= 0.875, else from n - 8.  Zero and subnormal m end
    // at the least e.
    const int n = (int)(m >> 23) - 126;
    int e = (m & 0x7fffffu) <= 0x600000u ? n - 9 : n - 8;
    e = e > -100 ? e : -100;
    const float inv = pow2(-e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inv, v[4 * i + 1] * inv, 0, false);
        codes[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inv, v[4 * i + 3] * inv, w, true);
    }
    return pow2(e);
}

struct Token {
    int64_t b, s, p;
};

EP_DEV Token token_at(const PagedTokens &t, uint32_t i)
{
    Token k;
    const uint32_t b = i / (uint32_t)t.S;
    k.b = b;
    k.s = i - b * (uint32_t)t.S;
    k.p = t.pos[k.b * t.pos_sb + k.s * t.pos_ss];
    __builtin_amdgcn_sched_barrier(0);      // ahead of the rows: what follows waits for it first
    return k;
}

// Which row a lane group of `lanes` works on: (token, head) of 256 / lanes
// rows a workgroup.
EP_DEV bool row_at(uint32_t rows, int heads, int lanes, uint32_t &token, int &head, int &u)
{
    const uint32_t r = blockIdx.x * (256u / lanes) + threadIdx.x / (uint32_t)lanes;
    u = threadIdx.x & (lanes - 1);
    if (r >= rows)
        return false;
    token = r / (uint32_t)heads;
    head = (int)(r - token * heads);
    return true;
}

struct RotateArgs {
    Rows q, k;
    Turn turn;
    PagedTokens tok;
    void *q_out, *k_out;
    uint32_t rows;
    int D, lanes;
};

template <typename T, bool VEC, bool STREAM>
__global__ void __launch_bounds__(256) rotate_kernel(RotateArgs a)
{
    uint32_t token;
    int head, u;
    if (!row_at(a.rows, a.q.heads + a.k.heads, a.lanes, token, head, u) || 16 * u >= a.D)
        return;
    const Token t = token_at(a.tok, token);
    const bool is_q = head < a.q.heads;
    const Rows x = pick(is_q, a.q, a.k);
    const int h = is_q ? head : head - a.q.heads;
    T *y = (T *)(is_q ? a.q_out : a.k_out) + ((int64_t)token * x.heads + h) * a.D;
    float v[16];
    LaneRow<T, VEC> row;
    row.load((const T *)x.ptr + t.b * x.sb + t.s * x.ss + h * x.sh, a.D, u, a.turn);
    const bool ok = t.p >= 0 && t.p < a.turn.max_pos;
    row.values(a.turn, ok, t.p, v);
    const float fill = t.p < 0 ? 0.0f : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int e = 0; e < 16; ++e)
        v[e] = ok ? v[e] : fill;
    store_row<VEC, STREAM>(y, a.D, row.ch, v);
}

struct AppendArgs {
    Rows q, k, v;
    Turn turn;
    PagedTokens tok;
    PagedCache c;
    void *q_out;
    uint32_t rows;
    int lanes;
};

// Position p's page and row in it; false (and the pool's first row, which can
// be read) for padding, past the table, or where the table names no page.
EP_DEV bool slot_of(const PagedTokens &t, const PagedCache &c, int64_t b, int64_t p, int64_t &page, int &row)
{
    const int64_t i = p >> c.page_shift;
    int32_t id = -1;
    if (p >= 0 && i < t.width)
        id = t.table[b * t.table_stride + i];
    const bool ok = id >= 0 && id < c.n_pages;
    page = ok ? id : 0;
    row = ok ? (int)(p & (c.page - 1)) : 0;
    return ok;
}

template <typename T, bool VEC, bool STREAM>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a)
{
    uint32_t token;
    int head, u;
    const int D = a.c.D, Hq = a.q.heads, Hk = a.c.heads;
    if (!row_at(a.rows, Hq + 2 * Hk, a.lanes, token, head, u))
        return;
    const Token t = token_at(a.tok, token);
    const bool mine = 16 * u < D;   // lanes past the row only take part in its maximum
    const bool is_q = head < Hq, is_v = head >= Hq + Hk;
    const Rows x = pick(is_q, a.q, pick(is_v, a.v, a.k));
    const int h = is_q ? head : is_v ? head - Hq - Hk : head - Hq;
    LaneRow<T, VEC> lane_row;       // lanes past the row take its start
    lane_row.load((const T *)x.ptr + t.b * x.sb + t.s * x.ss + h * x.sh, D, mine ? u : 0, a.turn);
    const Chunks ch = lane_row.ch;
    const bool turns = !is_v && a.turn.dim > 0;
    // one answer for a token's q, k and v: a value without its key is not stored either
    const bool known = t.p >= 0 && (a.turn.dim == 0 || t.p < a.turn.max_pos);
    int64_t page;
    int row;
    const bool stored = slot_of(a.tok, a.c, t.b, t.p, page, row);   // one answer for all lanes of a row
    float v[16];
    lane_row.values(a.turn, turns && known, t.p, v);
    const float fill = t.p < 0 || !mine ? 0.0f : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int e = 0; e < 16; ++e)
        v[e] = mine && known ? v[e] : fill;
    if (is_q) {
        if (mine)
            store_row<VEC, STREAM>((T *)a.q_out + ((int64_t)token * Hq + h) * D, D, ch, v);
        return;
    }
    if (!known || !stored)
        return;
    const int64_t at = (page * Hk + h) * a.c.page + row;
    void *dst = is_v ? a.c.v : a.c.k;
    if (a.c.dtype == EP_F16 || a.c.dtype == EP_BF16) {
        if (mine) {
            if (a.c.dtype == EP_F16)
                store_row<true, false>((f16_t *)dst + at * D, D, ch, v);
            else
                store_row<true, false>((uint16_t *)dst + at * D, D, ch, v);
        }
        return;
    }
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const uint32_t b = __float_as_uint(v[e]) & 0x7fffffffu;
        m = m > b ? m : b;
    }
    m = row_max(m, a.lanes);
    uint32_t codes[4];
    const float s = quantise(v, m, a.c.dtype, codes);
    if (mine) {
        uint8_t *p = (uint8_t *)dst + at * D;
        __builtin_memcpy(__builtin_assume_aligned(p + ch.a, 8), codes, 8);
        __builtin_memcpy(__builtin_assume_aligned(p + ch.b, 8), codes + 2, 8);
    }
    if (u == 0)
        (is_v ? a.c.v_scale : a.c.k_scale)[at] = s;
}

struct ReadArgs {
    PagedTokens tok;
    PagedCache c;
    void *k_out, *v_out;
    uint32_t rows;
    int lanes;
};

template <typename T, bool STREAM>
__global__ void __launch_bounds__(256) read_kernel(ReadArgs a)
{
    uint32_t token;
    int head, u;
    const int D = a.c.D, Hk = a.c.heads;
    if (!row_at(a.rows, 2 * Hk, a.lanes, token, head, u) || 16 * u >= D)
        return;
    const Token t = token_at(a.tok, token);
    const bool is_v = head >= Hk;
    const int h = is_v ? head - Hk : head;
    const Chunks ch = chunks_of(u, 0, D);
    int64_t page;
    int row;
    const bool ok = slot_of(a.tok, a.c, t.b, t.p, page, row);
    // Loaded either way, with no branch on ok: this compiler lost the value of
    // D that the output's address needs, in the lanes that skipped such a branch.
    const int64_t at = (page * Hk + h) * a.c.page + row;
    const void *src = is_v ? a.c.v : a.c.k;
    float v[16];
    if (a.c.dtype == EP_F16) {
        load8((const f16_t *)src + at * D + ch.a, v);
        load8((const f16_t *)src + at * D + ch.b, v + 8);
    } else if (a.c.dtype == EP_BF16) {
        load8((const uint16_t *)src + at * D + ch.a, v);
        load8((const uint16_t *)src + at * D + ch.b, v + 8);
    } else {
        const float s = (is_v ? a.c.v_scale : a.c.k_scale)[at];
        uint32_t w[4];
        __builtin_memcpy(w, __builtin_assume_aligned((const uint8_t *)src + at * D + ch.a, 8), 8);
        __builtin_memcpy(w + 2, __builtin_assume_aligned((const uint8_t *)src + at * D + ch.b, 8), 8);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            decode4(w[i], a.c.dtype, v + 4 * i);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            v[e] *= s;
    }
    const float fill = t.p < 0 ? 0.0f : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int e = 0; e < 16; ++e)
        v[e] = ok ? v[e] : fill;
    store_row<true, STREAM>((T *)(is_v ? a.v_out : a.k_out) + ((int64_t)token * Hk + h) * D, D, ch, v);
}

bool aligned(const void *p, int64_t n) { return ((uintptr_t)p % n) == 0; }

// A lane's chunks of these rows can be loaded whole.
bool whole_chunks(const ep_heads *x, int64_t B, int64_t S)
{
    const int n = x->dtype == EP_F32 ? 4 : 8;   // values in 16 bytes
    return aligned(x->ptr, 16) && (B == 1 || x->stride_b % n == 0) && (S == 1 || x->stride_s % n == 0) &&
           (x->heads == 1 || x->stride_h % n == 0);
}

int lanes_of(int64_t D)
{
    int n = 1;
    while (n * 16 < D)
        n *= 2;
    return n;
}

// D and the rotated part in whole chunks (in pairs of them where a lane's
// two chunks are the halves of its pairs, and the rest in 16s).
bool whole_rows(int64_t D, const ep_rotation *rot)
{
    return D % 16 == 0 && (!rot || (rot->dim % 16 == 0 && aligned(rot->cos_t, 16) && aligned(rot->sin_t, 16)));
}

Rows rows_of(const ep_heads *x)
{
    return x && x->ptr ? Rows{x->ptr, x->stride_b, x->stride_s, x->stride_h, x->heads} : Rows{nullptr, 0, 0, 0, 0};
}

Turn turn_of(const ep_rotation *rot, int inverse)
{
    if (!rot)
        return Turn{nullptr, nullptr, 0, 0, 0, 1.0f};
    return Turn{rot->cos_t, rot->sin_t, rot->max_pos, rot->dim, rot->interleaved, inverse ? -1.0f : 1.0f};
}

// More than half of what the L2 caches hold together: their inputs pass there too.
bool streams(int64_t values, int dtype) { return values * (dtype == EP_F32 ? 4 : 2) > (int64_t)16 << 20; }

// Rows of a call and its grid: a launch has fewer than 2^32 threads.
int grid_of(const PagedTokens &tok, int heads, int lanes, uint32_t &rows, unsigned &grid)
{
    const int64_t n = tok.B * tok.S * heads, per = 256 / lanes, groups = (n + per - 1) / per;
    if (groups > 0xffffff)
        return set_error(EP_DECLINE_SHAPE, "%lld rows on %d lanes each are more than one launch takes", (long long)n,
                         lanes);
    rows = (uint32_t)n;
    grid = (unsigned)groups;
    return EP_OK;
}

template <bool VEC, bool STREAM>
void rotate_typed(int dtype, unsigned grid, const RotateArgs &a, hipStream_t st)
{
    if (dtype == EP_F32)
        rotate_kernel<float, VEC, STREAM><<<grid, 256, 0, st>>>(a);
    else if (dtype == EP_F16)
        rotate_kernel<f16_t, VEC, STREAM><<<grid, 256, 0, st>>>(a);
    else
        rotate_kernel<uint16_t, VEC, STREAM><<<grid, 256, 0, st>>>(a);
}

template <bool VEC, bool STREAM>
void append_typed(int dtype, unsigned grid, const AppendArgs &a, hipStream_t st)
{
    if (dtype == EP_F32)
        append_kernel<float, VEC, STREAM><<<grid, 256, 0, st>>>(a);
    else if (dtype == EP_F16)
        append_kernel<f16_t, VEC, STREAM><<<grid, 256, 0, st>>>(a);
    else
        append_kernel<uint16_t, VEC, STREAM><<<grid, 256, 0, st>>>(a);
}

template <bool STREAM>
void read_typed(int dtype, unsigned grid, const ReadArgs &a, hipStream_t st)
{
    if (dtype == EP_F32)
        read_kernel<float, STREAM><<<grid, 256, 0, st>>>(a);
    else if (dtype == EP_F16)
        read_kernel<f16_t, STREAM><<<grid, 256, 0, st>>>(a);
    else
        read_kernel<uint16_t, STREAM><<<grid, 256, 0, st>>>(a);
}

}  // namespace

int launch_rotate(const ep_heads *q, const ep_heads *k, const ep_rotation *rot, const PagedTokens &tok, int64_t D,
                  int inverse, void *q_out, void *k_out, hipStream_t stream)
{
    RotateArgs a{rows_of(q), rows_of(k), turn_of(rot, inverse), tok, q_out, k_out, 0, (int)D, lanes_of(D)};
    unsigned grid;
    const int rc = grid_of(tok, a.q.heads + a.k.heads, a.lanes, a.rows, grid);
    if (rc != EP_OK || a.rows == 0)
        return rc;
    const bool vec = whole_rows(D, rot) && whole_chunks(q, tok.B, tok.S) && aligned(q_out, 16) &&
                     (!a.k.ptr || (whole_chunks(k, tok.B, tok.S) && aligned(k_out, 16)));
    if (vec && streams((int64_t)a.rows * D, q->dtype))
        rotate_typed<true, true>(q->dtype, grid, a, stream);
    else if (vec)
        rotate_typed<true, false>(q->dtype, grid, a, stream);
    else
        rotate_typed<false, false>(q->dtype, grid, a, stream);
    EP_HIP_CHECK(hipGetLastError());
    return EP_OK;
}

int launch_kv_append(const ep_heads *q, const ep_heads *k, const ep_heads *v, const ep_rotation *rot,
                     const PagedTokens &tok, const PagedCache &c, void *q_out, hipStream_t stream)
{
    AppendArgs a{rows_of(q), rows_of(k), rows_of(v), turn_of(rot, 0), tok, c, q_out, 0, lanes_of(c.D)};
    unsigned grid;
    const int rc = grid_of(tok, a.q.heads + 2 * c.heads, a.lanes, a.rows, grid);
    if (rc != EP_OK || a.rows == 0)
        return rc;
    const bool vec = whole_rows(c.D, rot) && whole_chunks(k, tok.B, tok.S) && whole_chunks(v, tok.B, tok.S) &&
                     (!a.q.ptr || (whole_chunks(q, tok.B, tok.S) && aligned(q_out, 16)));
    if (vec && streams(tok.B * tok.S * a.q.heads * c.D, k->dtype))
        append_typed<true, true>(k->dtype, grid, a, stream);
    else if (vec)
        append_typed<true, false>(k->dtype, grid, a, stream);
    else
        append_typed<false, false>(k->dtype, grid, a, stream);
    EP_HIP_CHECK(hipGetLastError());
    return EP_OK;
}

int launch_kv_read(const PagedTokens &tok, const PagedCache &c, void *k_out, void *v_out, int out_dtype,
                   hipStream_t stream)
{
    ReadArgs a{tok, c, k_out, v_out, 0, lanes_of(c.D)};
    unsigned grid;
    const int rc = grid_of(tok, 2 * c.heads, a.lanes, a.rows, grid);
    if (rc != EP_OK || a.rows == 0)
        return rc;
    if (!aligned(k_out, 16) || !aligned(v_out, 16))
        return set_error(EP_DECLINE_SHAPE, "cache read: outputs must be 16-byte aligned");
    if (streams((int64_t)a.rows * c.D, out_dtype))
        read_typed<true>(out_dtype, grid, a, stream);
    else
        read_typed<false>(out_dtype, grid, a, stream);
    EP_HIP_CHECK(hipGetLastError());
    return EP_OK;
}

}  // namespace ep
