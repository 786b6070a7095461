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
// reads x and dy and writes dx once. A row is held by L = D/16 lanes
// (rounded up to a power of two) with eight pairs each, so the rotation
// needs no exchange between lanes and the norm log2(L) shuffles. The rows
// of a wave are heads of one token: their angles are the same cache lines,
// read once and kept in registers over the heads.
#include "vec.hpp"

using namespace kfv;

namespace {

constexpr int BLOCK = 256;
constexpr int WAVES = BLOCK / WAVE;
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
    long long tokens;
    int S, D, lanes, lanes_log, wf32;
    float eps;
    int split, heads_per;   // waves that share a token, heads of each
    float *partial;         // backward: [blocks][2][D]
};

template <typename T, bool VEC>
__device__ inline void load_pairs(float *lo, float *hi, const T *row, int D,
                                  int li, int L)
{
    const int half = D / 2;
    if (VEC) {
        if (li * 8 < half) {
            ld8<T>(lo, row + li * 8);
            ld8<T>(hi, row + half + li * 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) lo[j] = hi[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = j * L + li;
            lo[j] = i < half ? (float)row[i] : 0.f;
            hi[j] = i < half ? (float)row[half + i] : 0.f;
        }
    }
}

template <typename T, bool VEC>
__device__ inline void store_pairs(T *row, const float *lo, const float *hi,
                                   int D, int li, int L)
{
    const int half = D / 2;
    if (VEC) {
        if (li * 8 < half) {
            st8<T>(row + li * 8, lo);
            st8<T>(row + half + li * 8, hi);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = j * L + li;
            if (i < half) {
                row[i] = (T)lo[j];
                row[half + i] = (T)hi[j];
            }
        }
    }
}

template <typename T, bool VEC>
__device__ inline void load_weight(float *lo, float *hi, const void *w,
                                   int wf32, int D, int li, int L)
{
    if (!w) {
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = hi[j] = 1.f;
    } else if (wf32) {
        load_pairs<float, VEC>(lo, hi, (const float *)w, D, li, L);
    } else {
        load_pairs<T, VEC>(lo, hi, (const T *)w, D, li, L);
    }
}

// cos and sin of this lane's pairs at token (b, s). A position outside the
// table is not followed: its angles, and so its rows, are NaN.
template <bool VEC>
__device__ inline void load_angles(float *cs, float *sn, const Args &a,
                                   int b, int s, int li)
{
    if (!a.rope) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cs[j] = 1.f;
            sn[j] = 0.f;
        }
        return;
    }
    long long pos = a.start + s;
    if (a.positions) {
        const long long at = b * a.pb + s * a.ps;
        pos = a.pwide ? ((const long long *)a.positions)[at]
                      : (long long)((const int *)a.positions)[at];
    }
    if (pos < 0 || pos >= a.P) {
#pragma unroll
        for (int j = 0; j < 8; ++j) cs[j] = sn[j] = __builtin_nanf("");
        return;
    }
    load_pairs<float, VEC>(cs, sn, a.rope + pos * a.D, a.D, li, a.lanes);
}

__device__ inline float group_sum(float v, int L)
{
    for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

template <typename T, bool VEC>
__device__ inline void fwd_rows(const Args &a, const Rows &x, int b, int s,
                                long long token, int h0, int h1, int li,
                                int gi, const float *cs, const float *sn)
{
    const int L = a.lanes, per = WAVE >> a.lanes_log;
    float wl[8], wh[8];
    load_weight<T, VEC>(wl, wh, x.w, a.wf32, a.D, li, L);
    for (int h = h0 + gi; h - gi < h1; h += per) {
        const bool on = h < h1;
        const T *row = (const T *)x.x + b * x.xb + s * x.xs +
                       (long long)(on ? h : h0) * x.xh;
        float lo[8], hi[8], yl[8], yh[8], q = 0.f;
        load_pairs<T, VEC>(lo, hi, row, a.D, li, L);
#pragma unroll
        for (int j = 0; j < 8; ++j) q += lo[j] * lo[j] + hi[j] * hi[j];
        const float r = rsqrtf(group_sum(q, L) / (float)a.D + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float u = lo[j] * r * wl[j], v = hi[j] * r * wh[j];
            yl[j] = u * cs[j] - v * sn[j];
            yh[j] = v * cs[j] + u * sn[j];
        }
        if (on)
            store_pairs<T, VEC>((T *)x.out + (token * x.heads + h) * a.D, yl,
                                yh, a.D, li, L);
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(BLOCK) void qk_fwd(Args a)
{
    const int lane = threadIdx.x % WAVE;
    const int li = lane & (a.lanes - 1), gi = lane >> a.lanes_log;
    const int all = a.q.heads + a.k.heads;
    const long long units = a.tokens * a.split;
    for (long long u = (long long)blockIdx.x * WAVES + threadIdx.x / WAVE;
         u < units; u += (long long)gridDim.x * WAVES) {
        const int token =
            __builtin_amdgcn_readfirstlane((int)(u / a.split));
        const int part =
            __builtin_amdgcn_readfirstlane((int)(u - (long long)token *
                                                         a.split));
        const int b = token / a.S, s = token - b * a.S;
        float cs[8], sn[8];
        load_angles<VEC>(cs, sn, a, b, s, li);
        const int h0 = part * a.heads_per;
        const int h1 = h0 + a.heads_per < all ? h0 + a.heads_per : all;
        if (h0 < a.q.heads)
            fwd_rows<T, VEC>(a, a.q, b, s, token, h0,
                             h1 < a.q.heads ? h1 : a.q.heads, li, gi, cs,
                             sn);
        if (h1 > a.q.heads)
            fwd_rows<T, VEC>(a, a.k, b, s, token,
                             h0 > a.q.heads ? h0 - a.q.heads : 0,
                             h1 - a.q.heads, li, gi, cs, sn);
    }
}

template <typename T, bool VEC>
__device__ inline void bwd_rows(const Args &a, const Rows &x, int b, int s,
                                long long token, int h0, int h1, int li,
                                int gi, const float *cs, const float *sn,
                                const float *wl, const float *wh, float *al,
                                float *ah)
{
    const int L = a.lanes, per = WAVE >> a.lanes_log;
    for (int h = h0 + gi; h - gi < h1; h += per) {
        const bool on = h < h1;
        const long long hh = on ? h : h0;
        float lo[8], hi[8], gl[8], gh[8], q = 0.f, t = 0.f;
        load_pairs<T, VEC>(lo, hi,
                           (const T *)x.x + b * x.xb + s * x.xs + hh * x.xh,
                           a.D, li, L);
        load_pairs<T, VEC>(gl, gh,
                           (const T *)x.dy + b * x.gb + s * x.gs + hh * x.gh,
                           a.D, li, L);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q += lo[j] * lo[j] + hi[j] * hi[j];
            const float u = gl[j] * cs[j] + gh[j] * sn[j];
            const float v = gh[j] * cs[j] - gl[j] * sn[j];
            gl[j] = u;
            gh[j] = v;
            t += u * wl[j] * lo[j] + v * wh[j] * hi[j];
        }
        const float r = rsqrtf(group_sum(q, L) / (float)a.D + a.eps);
        const float m = group_sum(t, L) / (float)a.D * r * r * r;
        if (on) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                al[j] += gl[j] * lo[j] * r;
                ah[j] += gh[j] * hi[j] * r;
                gl[j] = gl[j] * wl[j] * r - lo[j] * m;
                gh[j] = gh[j] * wh[j] * r - hi[j] * m;
            }
            store_pairs<T, VEC>((T *)x.out + (token * x.heads + h) * a.D, gl,
                                gh, a.D, li, L);
        }
    }
}

// Adds the row groups of every wave of the block in a fixed order and
// writes the block's sum of one weight's gradient.
template <bool VEC>
__device__ inline void block_weight(const float *al, const float *ah,
                                    float *lds, float *dst, int D, int li,
                                    int gi, int L, int per, int wid)
{
    const int half = D / 2;
    __syncthreads();
    float *mine = lds + wid * D;
    for (int g = 0; g < per; ++g) {  // a wave's groups, one after another
        if (g == gi) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = VEC ? li * 8 + j : j * L + li;
                if (i < half) {
                    mine[i] = (g ? mine[i] : 0.f) + al[j];
                    mine[half + i] = (g ? mine[half + i] : 0.f) + ah[j];
                }
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < D; i += BLOCK) {
        float v = 0.f;
        for (int w = 0; w < WAVES; ++w) v += lds[w * D + i];
        dst[i] = v;
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(BLOCK) void qk_bwd(Args a)
{
    __shared__ float lds[WAVES * MAX_D];
    const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
    const int li = lane & (a.lanes - 1), gi = lane >> a.lanes_log;
    const int all = a.q.heads + a.k.heads;
    const long long units = a.tokens * a.split;
    float qwl[8], qwh[8], kwl[8], kwh[8];
    float ql[8] = {}, qh[8] = {}, kl[8] = {}, kh[8] = {};
    load_weight<T, VEC>(qwl, qwh, a.q.w, a.wf32, a.D, li, a.lanes);
    load_weight<T, VEC>(kwl, kwh, a.k.w, a.wf32, a.D, li, a.lanes);
    for (long long u = (long long)blockIdx.x * WAVES + wid; u < units;
         u += (long long)gridDim.x * WAVES) {
        const int token =
            __builtin_amdgcn_readfirstlane((int)(u / a.split));
        const int part =
            __builtin_amdgcn_readfirstlane((int)(u - (long long)token *
                                                         a.split));
        const int b = token / a.S, s = token - b * a.S;
        float cs[8], sn[8];
        load_angles<VEC>(cs, sn, a, b, s, li);
        const int h0 = part * a.heads_per;
        const int h1 = h0 + a.heads_per < all ? h0 + a.heads_per : all;
        if (h0 < a.q.heads)
            bwd_rows<T, VEC>(a, a.q, b, s, token, h0,
                             h1 < a.q.heads ? h1 : a.q.heads, li, gi, cs,
                             sn, qwl, qwh, ql, qh);
        if (h1 > a.q.heads)
            bwd_rows<T, VEC>(a, a.k, b, s, token,
                             h0 > a.q.heads ? h0 - a.q.heads : 0,
                             h1 - a.q.heads, li, gi, cs, sn, kwl, kwh, kl,
                             kh);
    }
    if (a.partial) {
        float *dst = a.partial + (long long)blockIdx.x * 2 * a.D;
        const int per = WAVE >> a.lanes_log;
        block_weight<VEC>(ql, qh, lds, dst, a.D, li, gi, a.lanes, per, wid);
        block_weight<VEC>(kl, kh, lds, dst + a.D, a.D, li, gi, a.lanes, per,
                          wid);
    }
}

// dw[c] = sum of the blocks' partial sums, 64 columns a block: wave w adds
// every fourth partial, the four sums are added in order.
template <typename T>
__global__ __launch_bounds__(BLOCK) void qk_weight(
    const float *__restrict__ partial, int blocks, int D, int wf32,
    void *__restrict__ dqw, void *__restrict__ dkw)
{
    __shared__ float lds[WAVES][WAVE];
    const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
    const int c = blockIdx.x * WAVE + lane;
    float v = 0.f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int i = wid; i < blocks; i += WAVES)
            v += partial[(long long)i * 2 * D + c];
    }
    lds[wid][lane] = v;
    __syncthreads();
    if (wid == 0 && c < 2 * D) {
        v = lds[0][lane] + lds[1][lane] + lds[2][lane] + lds[3][lane];
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

// Heads of a token are shared by as many waves as keep four rows for each
// lane group, evenly.
void shape(Args &a)
{
    const int groups = (a.D / 2 + 7) / 8;
    a.lanes = 1;
    a.lanes_log = 0;
    while (a.lanes < groups) {
        a.lanes *= 2;
        a.lanes_log += 1;
    }
    const int all = a.q.heads + a.k.heads;
    const int most = 4 * (WAVE / a.lanes);
    a.split = (all + most - 1) / most;
    a.heads_per = (all + a.split - 1) / a.split;
}

constexpr int BWD_BLOCKS = 512;

long long blocks_of(const Args &a)
{
    return (a.tokens * a.split + WAVES - 1) / WAVES;
}

template <typename T>
hipError_t launch(Args &a, bool backward, void *dqw, void *dkw,
                  hipStream_t s)
{
    long long blocks = blocks_of(a);
    const bool vec = vec_ok(a, backward);
    if (!backward) {
        if (blocks > 1 << 20) blocks = 1 << 20;
        if (vec)
            qk_fwd<T, true><<<(unsigned)blocks, BLOCK, 0, s>>>(a);
        else
            qk_fwd<T, false><<<(unsigned)blocks, BLOCK, 0, s>>>(a);
        return hipGetLastError();
    }
    if (blocks > BWD_BLOCKS) blocks = BWD_BLOCKS;
    if (blocks < 1) blocks = 1;  // no tokens: the weights' zeros
    if (vec)
        qk_bwd<T, true><<<(unsigned)blocks, BLOCK, 0, s>>>(a);
    else
        qk_bwd<T, false><<<(unsigned)blocks, BLOCK, 0, s>>>(a);
    if (a.partial)
        qk_weight<T><<<(2 * a.D + WAVE - 1) / WAVE, BLOCK, 0, s>>>(
            a.partial, (int)blocks, a.D, a.wf32, dqw, dkw);
    return hipGetLastError();
}

}  // namespace

extern "C" {

// floats of the backward's workspace
long long kf_qk_ws(int D) { return (long long)BWD_BLOCKS * 2 * D; }

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
    a.tokens = dims[0];
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
    if (a.tokens < 0 || a.tokens >= 1ll << 30 || a.S < 1 || a.D < 2 ||
        a.D % 2 || a.D > MAX_D || a.q.heads < 0 || a.k.heads < 0 ||
        a.q.heads + a.k.heads < 1 || a.q.heads + a.k.heads > 1 << 16)
        return hipErrorInvalidValue;
    if (a.tokens == 0 && !a.partial) return hipSuccess;
    shape(a);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
    case 0: return launch<float>(a, backward, dqw, dkw, s);
    case 1: return launch<__bf16>(a, backward, dqw, dkw, s);
    case 2: return launch<_Float16>(a, backward, dqw, dkw, s);
    }
    return hipErrorInvalidValue;
}

}  // extern "C"
