// RMS norm of queries and keys for each head with the position rotation in
// the same pass — gfx950.
//
// For a head's row x of D elements, weight w and the angles a of its
// position (pairs are (i, i + D/2)):
//   r = rsqrt(mean(x^2) + eps)        u = x * r * w
//   y[i]       = u[i] cos a[i] - u[i + D/2] sin a[i]
//   y[i + D/2] = u[i + D/2] cos a[i] + u[i] sin a[i]
// Backward, with g = the inverse rotation of dy and h = g * w:
//   dw = sum over rows of g * x * r
//   dx = r * h - x * r^3 * mean(h * x)
// r is computed again from x, which the backward reads anyway.
//
// Both are bound by memory: forward reads x and writes y once, backward
// reads x and dy and writes dx once (2 x 8192 tokens, 32/8 heads of 128 in
// bf16: 335 MB in 63 us, 5.3 TB/s, and 503 MB in 117 us, 4.3 TB/s). A row
// is held by L = D/16 lanes (rounded up to a power of two) with eight pairs
// each, so the rotation needs no exchange between lanes and the norm log2(L)
// shuffles.
//
// A group of L lanes keeps one head and walks over the tokens, neighbouring
// groups are neighbouring heads of a token: what a group needs of the
// weights, and its sum of their gradient, stays in registers; the heads
// share the cache lines of their token's angles; and the group has the rows
// of several tokens on their way at once.
#include "vec.hpp"

using namespace kfv;

namespace {

constexpr int BLOCK = 256;
constexpr int MAX_D = 512;

struct Rows {          // [B][S][heads][D], last dimension dense
    const void *x;
    const void *dy;    // backward only
    void *out;         // dense [B][S][heads][D]: y, or dx
    long long xb, xs, xh, gb, gs, gh;
    const void *w;     // [D] or null
    int heads;
};

struct Args {
    Rows q, k;
    const float *rope;      // [P][D]: cos of D/2 angles, then sin; or null
    const void *positions;  // int64 or int32, [B][S] by strides; or null
    long long pb, ps;
    int pwide;
    long long start, P;
    int tokens, S, D, lanes, lanes_log, wf32;
    float eps;
    int groups, tstep;  // that have a head; tokens from one to the next
    float *partial;     // backward: [blocks][2][D]
};

// Eight pairs of a row, columns li * 8 + j (VEC) or j * L + li; columns
// past the last pair repeat one and are dropped.
template <bool VEC>
__device__ inline int pair_col(int li, int j, int L)
{
    return VEC ? li * 8 + j : j * L + li;
}

template <typename T, bool VEC>
struct Pairs {
    typename vec8<T>::type lo, hi;
    __device__ void load(const T *row, int half, int li, int L)
    {
        if (VEC) {
            const int c = li * 8 < half ? li * 8 : 0;
            lo = *(const typename vec8<T>::type *)(row + c);
            hi = *(const typename vec8<T>::type *)(row + half + c);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                int c = pair_col<VEC>(li, j, L);
                c = c < half ? c : 0;
                lo[j] = row[c];
                hi[j] = row[half + c];
            }
        }
    }
    // as f32; zeros past the last pair
    __device__ void get(float *l, float *h, int half, int li, int L) const
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = (VEC ? li * 8 : pair_col<VEC>(li, j, L)) < half;
            l[j] = in ? (float)lo[j] : 0.f;
            h[j] = in ? (float)hi[j] : 0.f;
        }
    }
};

template <typename T, bool VEC>
__device__ inline void store_pairs(T *row, const float *lo, const float *hi,
                                   int half, int li, int L)
{
    if (VEC) {
        if (li * 8 < half) {
            st8<T>(row + li * 8, lo);
            st8<T>(row + half + li * 8, hi);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = pair_col<VEC>(li, j, L);
            if (i < half) {
                row[i] = (T)lo[j];
                row[half + i] = (T)hi[j];
            }
        }
    }
}

template <typename T, bool VEC>
__device__ inline void load_weight(float *lo, float *hi, const void *w,
                                   int wf32, int half, int li, int L)
{
    if (!w) {
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = hi[j] = 1.f;
    } else if (wf32) {
        Pairs<float, VEC> p;
        p.load((const float *)w, half, li, L);
        p.get(lo, hi, half, li, L);
    } else {
        Pairs<T, VEC> p;
        p.load((const T *)w, half, li, L);
        p.get(lo, hi, half, li, L);
    }
}

__device__ inline float group_sum(float v, int L)
{
    for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// A lane group's way over the tokens: its head, and where its rows of the
// token it stands at begin. Past the last token it stands still.
template <typename T, bool BWD>
struct Walk {
    int token, b, s;
    const T *x, *dy;
    T *out;
    long long step_x, wrap_x, step_g, wrap_g, step_o;
    bool is_q;
    __device__ Walk(const Args &a, int gid)
    {
        const int all = a.q.heads + a.k.heads;
        token = gid / all;
        int h = gid - token * all;
        if (gid >= a.groups) token = a.tokens;
        is_q = h < a.q.heads;
        const Rows &r = is_q ? a.q : a.k;
        h = is_q ? h : h - a.q.heads;
        const int t = token < a.tokens ? token : 0;
        b = t / a.S;
        s = t - b * a.S;
        const int db = a.tstep / a.S, ds = a.tstep - db * a.S;
        const long long xb = is_q ? a.q.xb : a.k.xb;
        const long long xs = is_q ? a.q.xs : a.k.xs;
        const long long xh = is_q ? a.q.xh : a.k.xh;
        x = (const T *)(is_q ? a.q.x : a.k.x) + b * xb + s * xs + h * xh;
        step_x = db * xb + ds * xs;
        wrap_x = xb - a.S * xs;
        const int heads = is_q ? a.q.heads : a.k.heads;
        out = (T *)(is_q ? a.q.out : a.k.out) +
              ((long long)t * heads + h) * a.D;
        step_o = (long long)a.tstep * heads * a.D;
        if (BWD) {
            const long long gb = is_q ? a.q.gb : a.k.gb;
            const long long gs = is_q ? a.q.gs : a.k.gs;
            const long long gh = is_q ? a.q.gh : a.k.gh;
            dy = (const T *)(is_q ? a.q.dy : a.k.dy) + b * gb + s * gs +
                 h * gh;
            step_g = db * gb + ds * gs;
            wrap_g = gb - a.S * gs;
        }
    }
    __device__ bool on(const Args &a) const { return token < a.tokens; }
    __device__ void next(const Args &a)
    {
        if (token < a.tokens - a.tstep) {
            const int db = a.tstep / a.S, ds = a.tstep - db * a.S;
            b += db;
            s += ds;
            x += step_x;
            out += step_o;
            if (BWD) dy += step_g;
            if (s >= a.S) {
                s -= a.S;
                b += 1;
                x += wrap_x;
                if (BWD) dy += wrap_g;
            }
            token += a.tstep;
        } else {
            token = a.tokens;
        }
    }
    // Row of the table; -1 for a position outside it, which is not
    // followed: its rows are NaN and have no gradient.
    __device__ long long position(const Args &a) const
    {
        long long pos = a.start + s;
        if (a.positions) {
            const long long at = b * a.pb + s * a.ps;
            pos = a.pwide ? ((const long long *)a.positions)[at]
                          : (long long)((const int *)a.positions)[at];
        }
        return pos < 0 || pos >= a.P ? -1 : pos;
    }
};

template <typename T, bool VEC>
struct Angles {
    Pairs<float, VEC> p;
    bool ok;
    template <typename W>
    __device__ void load(const Args &a, const W &w, int li)
    {
        ok = true;
        if (!a.rope) return;
        const long long pos = w.position(a);
        ok = pos >= 0;
        p.load(a.rope + (ok ? pos : 0) * a.D, a.D / 2, li, a.lanes);
    }
    __device__ void get(float *cs, float *sn, const Args &a) const
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cs[j] = !a.rope ? 1.f : ok ? p.lo[j] : __builtin_nanf("");
            sn[j] = !a.rope ? 0.f : ok ? p.hi[j] : __builtin_nanf("");
        }
    }
};

// U tokens at a time: their loads go out together.
template <typename T, bool VEC, int U>
__global__ __launch_bounds__(BLOCK) void qk_fwd(const Args a)
{
    const int lane = threadIdx.x % WAVE;
    const int L = a.lanes, li = lane & (L - 1), half = a.D / 2;
    Walk<T, false> w(a, (blockIdx.x * BLOCK + threadIdx.x) >> a.lanes_log);
    float wl[8], wh[8];
    load_weight<T, VEC>(wl, wh, w.is_q ? a.q.w : a.k.w, a.wf32, half, li, L);
    const int turns = (a.tokens + a.tstep - 1) / a.tstep;
    for (int turn = 0; turn < turns; turn += U) {
        Pairs<T, VEC> x[U];
        Angles<T, VEC> ang[U];
        T *out[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            on[u] = w.on(a);
            out[u] = w.out;
            x[u].load(w.x, half, li, L);
            ang[u].load(a, w, li);
            w.next(a);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float lo[8], hi[8], cs[8], sn[8], q = 0.f;
            x[u].get(lo, hi, half, li, L);
            ang[u].get(cs, sn, a);
#pragma unroll
            for (int j = 0; j < 8; ++j) q += lo[j] * lo[j] + hi[j] * hi[j];
            const float r = rsqrtf(group_sum(q, L) / (float)a.D + a.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float c = lo[j] * r * wl[j], d = hi[j] * r * wh[j];
                lo[j] = c * cs[j] - d * sn[j];
                hi[j] = d * cs[j] + c * sn[j];
            }
            if (on[u]) store_pairs<T, VEC>(out[u], lo, hi, half, li, L);
        }
    }
}

template <typename T, bool VEC, int U>
__global__ __launch_bounds__(BLOCK) void qk_bwd(const Args a)
{
    __shared__ float lds[BLOCK * 16];  // [groups][D]
    const int lane = threadIdx.x % WAVE;
    const int L = a.lanes, li = lane & (L - 1), half = a.D / 2;
    Walk<T, true> w(a, (blockIdx.x * BLOCK + threadIdx.x) >> a.lanes_log);
    float wl[8], wh[8], al[8] = {}, ah[8] = {};
    load_weight<T, VEC>(wl, wh, w.is_q ? a.q.w : a.k.w, a.wf32, half, li, L);
    const int turns = (a.tokens + a.tstep - 1) / a.tstep;
    for (int turn = 0; turn < turns; turn += U) {
        Pairs<T, VEC> x[U], dy[U];
        Angles<T, VEC> ang[U];
        T *out[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            on[u] = w.on(a);
            out[u] = w.out;
            x[u].load(w.x, half, li, L);
            dy[u].load(w.dy, half, li, L);
            ang[u].load(a, w, li);
            w.next(a);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float lo[8], hi[8], gl[8], gh[8], cs[8], sn[8];
            float q = 0.f, t = 0.f;
            x[u].get(lo, hi, half, li, L);
            dy[u].get(gl, gh, half, li, L);
            ang[u].get(cs, sn, a);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                q += lo[j] * lo[j] + hi[j] * hi[j];
                const float c = gl[j] * cs[j] + gh[j] * sn[j];
                const float d = gh[j] * cs[j] - gl[j] * sn[j];
                gl[j] = c;
                gh[j] = d;
                t += c * wl[j] * lo[j] + d * wh[j] * hi[j];
            }
            const float r = rsqrtf(group_sum(q, L) / (float)a.D + a.eps);
            const float m = group_sum(t, L) / (float)a.D * r * r * r;
            if (on[u] && ang[u].ok) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    al[j] += gl[j] * lo[j] * r;
                    ah[j] += gh[j] * hi[j] * r;
                    gl[j] = gl[j] * wl[j] * r - lo[j] * m;
                    gh[j] = gh[j] * wh[j] * r - hi[j] * m;
                }
                store_pairs<T, VEC>(out[u], gl, gh, half, li, L);
            } else if (on[u]) {
                // a row at a position outside the table has no gradient,
                // whatever it holds: zeros, and no part in the weights'
                const float zero[8] = {};
                store_pairs<T, VEC>(out[u], zero, zero, half, li, L);
            }
        }
    }
    if (!a.partial) return;
    // the block's sums: its groups' in order, q's and k's apart
    const int g = threadIdx.x >> a.lanes_log;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int i = pair_col<VEC>(li, j, L);
        if (i < half) {
            lds[g * a.D + i] = al[j];
            lds[g * a.D + half + i] = ah[j];
        }
    }
    __syncthreads();
    const int all = a.q.heads + a.k.heads, groups = BLOCK >> a.lanes_log;
    const int h0 = (int)((long long)blockIdx.x * groups % all);
    float *dst = a.partial + (long long)blockIdx.x * 2 * a.D;
    for (int i = threadIdx.x; i < 2 * a.D; i += BLOCK) {
        const bool want_q = i < a.D;
        const int c = want_q ? i : i - a.D;
        float v = 0.f;
        for (int k = 0, h = h0; k < groups; ++k) {
            if ((h < a.q.heads) == want_q) v += lds[k * a.D + c];
            h = h + 1 < all ? h + 1 : 0;
        }
        dst[i] = v;
    }
}

// dw[c] = sum of the blocks' partial sums, 64 columns a block: each of 16
// waves adds every 16th partial, the waves' sums are added in order.
constexpr int WBLOCK = 1024;
template <typename T>
__global__ __launch_bounds__(WBLOCK) void qk_weight(
    const float *__restrict__ partial, int blocks, int D, int wf32,
    void *__restrict__ dqw, void *__restrict__ dkw)
{
    constexpr int NW = WBLOCK / WAVE;
    __shared__ float lds[NW][WAVE];
    const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
    const int c = blockIdx.x * WAVE + lane;
    float v = 0.f;
    if (c < 2 * D) {
#pragma unroll 16
        for (int i = wid; i < blocks; i += NW)
            v += partial[(long long)i * 2 * D + c];
    }
    lds[wid][lane] = v;
    __syncthreads();
    if (wid == 0 && c < 2 * D) {
        v = 0.f;
        for (int i = 0; i < NW; ++i) v += lds[i][lane];
        void *dw = c < D ? dqw : dkw;
        const int i = c < D ? c : c - D;
        if (dw) {
            if (wf32)
                ((float *)dw)[i] = v;
            else
                ((T *)dw)[i] = (T)v;
        }
    }
}

bool vec_ok(const Args &a, bool backward)
{
    bool ok = a.D % 16 == 0 && aligned16(a.rope);
    for (const Rows *r : {&a.q, &a.k}) {
        ok = ok && aligned16(r->x) && aligned16(r->out) &&
             aligned16(r->w) &&
             ((r->xb | r->xs | r->xh) & 7) == 0;
        if (backward)
            ok = ok && aligned16(r->dy) &&
                 ((r->gb | r->gs | r->gh) & 7) == 0;
    }
    return ok;
}

constexpr int FWD_U = 2, BWD_U = 2;  // rows of a group on their way
constexpr int FWD_BLOCKS = 1024, BWD_BLOCKS = 512;

// Lanes of a row, and blocks: a group for each head of as many tokens as
// leave each group U rows, up to as many blocks as the chip holds.
int shape(Args &a, int U, int most)
{
    const int need = (a.D / 2 + 7) / 8;
    a.lanes = 1;
    a.lanes_log = 0;
    while (a.lanes < need) {
        a.lanes *= 2;
        a.lanes_log += 1;
    }
    const long long all = a.q.heads + a.k.heads;
    const long long per = BLOCK / a.lanes;  // groups of a block
    long long blocks =
        (all * ((a.tokens + U - 1) / U) + per - 1) / per;
    if (blocks > most) blocks = most;
    const long long least = (all + per - 1) / per;
    if (blocks < least) blocks = least;
    long long tstep = blocks * per / all;
    if (tstep > a.tokens) tstep = a.tokens > 0 ? a.tokens : 1;
    a.tstep = (int)tstep;
    a.groups = (int)(tstep * all);
    return (int)blocks;
}

template <typename T>
hipError_t launch(Args &a, bool backward, void *dqw, void *dkw,
                  hipStream_t s)
{
    const bool vec = vec_ok(a, backward);
    if (!backward) {
        const int blocks = shape(a, FWD_U, FWD_BLOCKS);
        if (vec)
            qk_fwd<T, true, FWD_U><<<blocks, BLOCK, 0, s>>>(a);
        else
            qk_fwd<T, false, FWD_U><<<blocks, BLOCK, 0, s>>>(a);
        return hipGetLastError();
    }
    const int blocks = shape(a, BWD_U, BWD_BLOCKS);
    if (vec)
        qk_bwd<T, true, BWD_U><<<blocks, BLOCK, 0, s>>>(a);
    else
        qk_bwd<T, false, BWD_U><<<blocks, BLOCK, 0, s>>>(a);
    if (a.partial)
        qk_weight<T><<<(2 * a.D + WAVE - 1) / WAVE, WBLOCK, 0, s>>>(
            a.partial, blocks, a.D, a.wf32, dqw, dkw);
    return hipGetLastError();
}

}  // namespace

extern "C" {

// floats of the backward's workspace
long long kf_qk_ws(int D, int heads)
{
    Args a = {};
    a.D = D;
    a.q.heads = heads;
    a.tokens = 1 << 30;
    return (long long)shape(a, BWD_U, BWD_BLOCKS) * 2 * D;
}

// ptrs: q, k, qw, kw, out_q, out_k, rope, positions
//       [, dyq, dyk, dqw, dkw, partial]
// dims: tokens, S, D, q heads, k heads, q strides (b s h), k strides,
//       P, start, positions strides (b s), positions are int64, w is f32
//       [, dyq strides, dyk strides]
hipError_t kf_qk_norm_rope(const uintptr_t *ptrs, const long long *dims,
                           int dtype, float eps, int backward, void *stream)
{
    Args a = {};
    a.q.x = (const void *)ptrs[0];
    a.k.x = (const void *)ptrs[1];
    a.q.w = (const void *)ptrs[2];
    a.k.w = (const void *)ptrs[3];
    a.q.out = (void *)ptrs[4];
    a.k.out = (void *)ptrs[5];
    a.rope = (const float *)ptrs[6];
    a.positions = (const void *)ptrs[7];
    if (dims[0] < 0 || dims[0] >= 1ll << 30 || dims[1] < 1 ||
        dims[1] >= 1ll << 30 || dims[2] < 2 || dims[2] > MAX_D ||
        dims[2] % 2 || dims[3] < 0 || dims[4] < 0 ||
        dims[3] + dims[4] < 1 || dims[3] + dims[4] > 1 << 16)
        return hipErrorInvalidValue;
    a.tokens = (int)dims[0];
    a.S = (int)dims[1];
    a.D = (int)dims[2];
    a.q.heads = (int)dims[3];
    a.k.heads = (int)dims[4];
    a.q.xb = dims[5];
    a.q.xs = dims[6];
    a.q.xh = dims[7];
    a.k.xb = dims[8];
    a.k.xs = dims[9];
    a.k.xh = dims[10];
    a.P = dims[11];
    a.start = dims[12];
    a.pb = dims[13];
    a.ps = dims[14];
    a.pwide = (int)dims[15];
    a.wf32 = (int)dims[16];
    a.eps = eps;
    void *dqw = nullptr, *dkw = nullptr;
    if (backward) {
        a.q.dy = (const void *)ptrs[8];
        a.k.dy = (const void *)ptrs[9];
        dqw = (void *)ptrs[10];
        dkw = (void *)ptrs[11];
        a.partial = (float *)ptrs[12];
        a.q.gb = dims[17];
        a.q.gs = dims[18];
        a.q.gh = dims[19];
        a.k.gb = dims[20];
        a.k.gs = dims[21];
        a.k.gh = dims[22];
    }
    if (a.tokens == 0 && !a.partial) return hipSuccess;
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
    case 0: return launch<float>(a, backward, dqw, dkw, s);
    case 1: return launch<__bf16>(a, backward, dqw, dkw, s);
    case 2: return launch<_Float16>(a, backward, dqw, dkw, s);
    }
    return hipErrorInvalidValue;
}

}  // extern "C"
