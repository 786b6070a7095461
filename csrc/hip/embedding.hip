// Embedding lookup with a scale, and its gradient by sorted tokens — gfx950.
//
//   out[n] = round(scale * W[ids[n]])
//   dW[v]  = round(scale * sum of dout[n] over n with ids[n] == v)
//
// The gradient is dense, so its floor is one read of dout and one write of
// dW. Atomic adds into dW would make the sum's order, and so its bits,
// change from run to run; here the ids are sorted by a stable radix sort
// and each row of dW is summed in one fixed order in f32, then scaled and
// rounded once.
//
// An id outside [0, V) is not followed: its output row is NaN and it
// adds to no gradient. The same key (V, the largest) takes the padding id
// out of the gradient.
#include "vec.hpp"

using namespace kfv;

namespace {

constexpr int BLOCK = 256;
constexpr int SORT_TILE = 4096;           // keys a block ranks in one pass
constexpr int SORT_ROUNDS = SORT_TILE / BLOCK;
constexpr int WAVES = BLOCK / WAVE;
constexpr int MAX_BITS = 8;               // digit bits of one pass
constexpr int MAX_DIGITS = 1 << MAX_BITS;
constexpr int CHUNK = 32;                 // rows that one partial sum joins
constexpr int COLS = WAVE * 8;            // columns that one wave sums

__device__ inline unsigned load_key(const void *ids, int wide, long long n,
                                    long long V, long long padding)
{
    const long long id = wide ? ((const long long *)ids)[n]
                              : (long long)((const int *)ids)[n];
    return id < 0 || id >= V || id == padding ? (unsigned)V : (unsigned)id;
}

// ---- forward ----
// A block takes `rows` consecutive ids; its threads run over their vectors
// of eight columns (VEC) or their columns one by one (rows that are not
// 16-byte aligned), so that neighbours always touch neighbouring bytes.
template <typename W, typename O, bool VEC>
__global__ __launch_bounds__(BLOCK) void embed_fwd(
    const void *__restrict__ ids, int wide, const W *__restrict__ weight,
    long long ldw, O *__restrict__ out, long long N, long long V, int H,
    int rows, float scale)
{
    const int per = VEC ? H / 8 : H;
    for (long long n0 = (long long)blockIdx.x * rows; n0 < N;
         n0 += (long long)gridDim.x * rows) {
        const int here = (int)(N - n0 < rows ? N - n0 : rows);
        for (int i = threadIdx.x; i < here * per; i += BLOCK) {
            const int r = i / per, c = i - r * per;
            const long long id = wide ? ((const long long *)ids)[n0 + r]
                                      : (long long)((const int *)ids)[n0 + r];
            const bool ok = id >= 0 && id < V;
            if (VEC) {
                float f[8];
                if (ok) {
                    ld8<W>(f, weight + id * ldw + c * 8);
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] *= scale;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = __builtin_nanf("");
                }
                st8<O>(out + (n0 + r) * H + c * 8, f);
            } else {
                const float f = ok ? (float)weight[id * ldw + c] * scale
                                   : __builtin_nanf("");
                out[(n0 + r) * H + c] = (O)f;
            }
        }
    }
}

// ---- stable radix sort of (token, position), least digit first ----
// One pass: hist counts the digits of each tile, scan turns the counts
// (digit-major) into first places, scatter ranks the keys of a tile in
// order and moves them. FIRST reads the ids themselves.
template <bool FIRST>
__global__ __launch_bounds__(BLOCK) void sort_hist(
    const void *__restrict__ src, int wide, long long N, long long V,
    long long padding, int shift, int bits, unsigned *__restrict__ hist,
    int nb, int *__restrict__ spans)
{
    __shared__ unsigned cnt[MAX_DIGITS];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    if (FIRST)  // no token has rows until bounds finds them
        for (long long i = (long long)blockIdx.x * BLOCK + threadIdx.x;
             i < 2 * V; i += (long long)gridDim.x * BLOCK)
            spans[i] = 0;
    const long long base = (long long)blockIdx.x * SORT_TILE;
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * BLOCK + threadIdx.x;
        if (n < N) {
            const unsigned key =
                FIRST ? load_key(src, wide, n, V, padding)
                      : ((const unsigned *)src)[n];
            atomicAdd(&cnt[(key >> shift) & ((1u << bits) - 1)], 1u);
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < 1 << bits)
        hist[(long long)threadIdx.x * nb + blockIdx.x] = cnt[threadIdx.x];
}

// Exclusive prefix sum of `n` counts by one block.
__global__ __launch_bounds__(1024) void sort_scan(unsigned *__restrict__ hist,
                                                  int n)
{
    __shared__ unsigned wsum[1024 / WAVE];
    const int lane = threadIdx.x % WAVE, w = threadIdx.x / WAVE;
    unsigned carry = 0;
    for (int base = 0; base < n; base += 1024 * 4) {
        const int i0 = base + (int)threadIdx.x * 4;
        unsigned v[4], s = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = i0 + j < n ? hist[i0 + j] : 0;
            s += v[j];
        }
        unsigned inc = s;
        for (int off = 1; off < WAVE; off <<= 1) {
            const unsigned t = __shfl_up(inc, off);
            if (lane >= off) inc += t;
        }
        if (lane == WAVE - 1) wsum[w] = inc;
        __syncthreads();
        unsigned before = carry, all = 0;
        for (int k = 0; k < 1024 / WAVE; ++k) {
            if (k < w) before += wsum[k];
            all += wsum[k];
        }
        before += inc - s;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i0 + j < n) hist[i0 + j] = before;
            before += v[j];
        }
        carry += all;
        __syncthreads();
    }
}

template <bool FIRST>
__global__ __launch_bounds__(BLOCK) void sort_scatter(
    const void *__restrict__ src, int wide,
    const unsigned *__restrict__ src_pos, long long N, long long V,
    long long padding, int shift, int bits,
    const unsigned *__restrict__ place, int nb, unsigned *__restrict__ dst,
    unsigned *__restrict__ dst_pos)
{
    // keys of one wave lie together, so wave order is key order
    __shared__ unsigned cnt[WAVES][MAX_DIGITS];
    const int lane = threadIdx.x % WAVE, w = threadIdx.x / WAVE;
    for (int i = threadIdx.x; i < WAVES * MAX_DIGITS; i += BLOCK)
        (&cnt[0][0])[i] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * SORT_TILE +
                           w * (SORT_TILE / WAVES) + lane;
    unsigned key[SORT_ROUNDS], rank[SORT_ROUNDS];
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * WAVE;
        key[r] = n >= N ? 0u
                 : FIRST ? load_key(src, wide, n, V, padding)
                         : ((const unsigned *)src)[n];
    }
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const bool in = base + r * WAVE < N;
        const unsigned d = (key[r] >> shift) & ((1u << bits) - 1);
        // lanes with the same digit
        unsigned long long same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long one = __ballot((d >> b) & 1);
            same &= (d >> b) & 1 ? one : ~one;
        }
        const unsigned before = __builtin_popcountll(
            same & ((1ull << lane) - 1));
        rank[r] = *(volatile unsigned *)&cnt[w][d] + before;
        __builtin_amdgcn_wave_barrier();
        if (in && before == 0)
            *(volatile unsigned *)&cnt[w][d] =
                rank[r] + __builtin_popcountll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d < 1 << bits) {
        unsigned at = place[(long long)d * nb + blockIdx.x];
        for (int k = 0; k < WAVES; ++k) {
            const unsigned c = cnt[k][d];
            cnt[k][d] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * WAVE;
        if (n < N) {
            const unsigned to =
                cnt[w][(key[r] >> shift) & ((1u << bits) - 1)] + rank[r];
            dst[to] = key[r];
            dst_pos[to] = FIRST ? (unsigned)n : src_pos[n];
        }
    }
}

// spans[v] = {first, one past the last} place of token v
__global__ __launch_bounds__(BLOCK) void token_bounds(
    const unsigned *__restrict__ keys, long long N, unsigned V,
    int *__restrict__ spans)
{
    const long long n = (long long)blockIdx.x * BLOCK + threadIdx.x;
    if (n >= N) return;
    const unsigned k = keys[n];
    if (k >= V) return;
    if (n == 0 || keys[n - 1] != k) spans[2 * (long long)k] = (int)n;
    if (n == N - 1 || keys[n + 1] != k) spans[2 * (long long)k + 1] = (int)n + 1;
}

// Columns of lane `lane`: eight neighbours (VEC), or every 64th.
template <bool VEC>
__device__ inline int col_of(int c0, int lane, int j)
{
    return VEC ? c0 + lane * 8 + j : c0 + j * WAVE + lane;
}

template <typename T, bool VEC>
__device__ inline void add_row(float *acc, const T *row, int c0, int lane,
                               int H)
{
    if (VEC) {
        if (c0 + lane * 8 < H) {
            float f[8];
            ld8<T>(f, row + c0 + lane * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += f[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<VEC>(c0, lane, j);
            if (c < H) acc[j] += (float)row[c];
        }
    }
}

// Sums of CHUNK neighbours of the sorted order that belong to one token,
// so that a frequent token's row is not one long chain of reads. Level 1
// sums rows of dout, level 2 sums level 1's results.
template <typename T, bool VEC, int LEVEL>
__global__ __launch_bounds__(BLOCK) void embed_partial(
    const unsigned *__restrict__ keys, const unsigned *__restrict__ pos,
    const T *__restrict__ dout, const float *__restrict__ part1,
    float *__restrict__ part, long long N, unsigned V, int H, int slices)
{
    const int lane = threadIdx.x % WAVE;
    const long long unit = __builtin_amdgcn_readfirstlane(
        (int)(blockIdx.x * WAVES + threadIdx.x / WAVE));
    const long long chunk = unit / slices;
    const int c0 = (int)(unit - chunk * slices) * COLS;
    constexpr int SPAN = LEVEL == 1 ? CHUNK : CHUNK * CHUNK;
    const long long i0 = chunk * SPAN;
    if (i0 + SPAN > N) return;
    const unsigned k = keys[i0];
    if (k >= V || keys[i0 + SPAN - 1] != k) return;
    float acc[8] = {};
#pragma unroll 8
    for (int i = 0; i < CHUNK; ++i) {
        if (LEVEL == 1)
            add_row<T, VEC>(acc, dout + (long long)pos[i0 + i] * H, c0,
                            lane, H);
        else
            add_row<float, VEC>(acc, part1 + (chunk * CHUNK + i) * H, c0,
                                lane, H);
    }
    float *row = part + chunk * H;
    if (VEC) {
        if (c0 + lane * 8 < H) st8<float>(row + c0 + lane * 8, acc);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<VEC>(c0, lane, j);
            if (c < H) row[c] = acc[j];
        }
    }
}

// One wave writes 512 columns of one row of dW: zeros, or the token's rows
// in their order, whole chunks by their partial sums.
template <typename T, typename W, bool VEC>
__global__ __launch_bounds__(BLOCK) void embed_rows(
    const int *__restrict__ spans, const unsigned *__restrict__ pos,
    const T *__restrict__ dout, const float *__restrict__ part1,
    const float *__restrict__ part2, W *__restrict__ dw, long long units,
    int H, int slices, float scale)
{
    const int lane = threadIdx.x % WAVE;
    for (long long u = (long long)blockIdx.x * WAVES + threadIdx.x / WAVE;
         u < units; u += (long long)gridDim.x * WAVES) {
        const int v = __builtin_amdgcn_readfirstlane((int)(u / slices));
        const int c0 = __builtin_amdgcn_readfirstlane(
            (int)(u - (long long)v * slices) * COLS);
        int i = spans[2 * (long long)v];
        const int end = spans[2 * (long long)v + 1];
        float acc[8] = {};
        while (i < end) {
            if (i % CHUNK == 0 && end - i >= CHUNK) {
                constexpr int BIG = CHUNK * CHUNK;
                if (i % BIG == 0 && end - i >= BIG) {
                    add_row<float, VEC>(acc, part2 + (long long)(i / BIG) * H,
                                        c0, lane, H);
                    i += BIG;
                } else {
                    add_row<float, VEC>(acc,
                                        part1 + (long long)(i / CHUNK) * H,
                                        c0, lane, H);
                    i += CHUNK;
                }
            } else {
                add_row<T, VEC>(acc, dout + (long long)pos[i] * H, c0, lane,
                                H);
                i += 1;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] *= scale;
        W *row = dw + (long long)v * H;
        if (VEC) {
            if (c0 + lane * 8 < H) st8<W>(row + c0 + lane * 8, acc);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = col_of<VEC>(c0, lane, j);
                if (c < H) row[c] = (W)acc[j];
            }
        }
    }
}

inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

struct Workspace {
    unsigned *keys[2], *pos[2], *hist;
    int *spans;
    float *part1, *part2;
    size_t bytes;
    Workspace(char *p, long long N, long long V, int H)
    {
        const long long nb = N / SORT_TILE + 1;
        size_t at = 0;
        auto take = [&](size_t n) {
            char *q = p + at;
            at += up256(n);
            return q;
        };
        for (int i = 0; i < 2; ++i) {
            keys[i] = (unsigned *)take(N * 4);
            pos[i] = (unsigned *)take(N * 4);
        }
        hist = (unsigned *)take(nb * MAX_DIGITS * 4);
        spans = (int *)take(V * 8);
        part1 = (float *)take((size_t)(N / CHUNK) * H * 4);
        part2 = (float *)take((size_t)(N / (CHUNK * CHUNK)) * H * 4);
        bytes = at;
    }
};

template <typename W, typename O>
hipError_t fwd(const void *ids, int wide, const void *weight, long long ldw,
               void *out, long long N, long long V, int H, float scale,
               hipStream_t s)
{
    const bool vec = H % 8 == 0 && ldw % 8 == 0 && aligned16(weight) &&
                     aligned16(out);
    const int per = vec ? H / 8 : H;
    // about four vectors a thread
    const int rows = per >= 4 * BLOCK ? 1 : 4 * BLOCK / per;
    long long blocks = (N + rows - 1) / rows;
    if (blocks > 1 << 20) blocks = 1 << 20;
    if (vec)
        embed_fwd<W, O, true><<<(unsigned)blocks, BLOCK, 0, s>>>(
            ids, wide, (const W *)weight, ldw, (O *)out, N, V, H, rows,
            scale);
    else
        embed_fwd<W, O, false><<<(unsigned)blocks, BLOCK, 0, s>>>(
            ids, wide, (const W *)weight, ldw, (O *)out, N, V, H, rows,
            scale);
    return hipGetLastError();
}

template <typename T, typename W, bool VEC>
hipError_t sums(const Workspace &ws, int at, const void *dout, void *dw,
                long long N, long long V, int H, float scale, hipStream_t s)
{
    const int slices = (H + COLS - 1) / COLS;
    const long long n1 = N / CHUNK * slices;
    if (n1)
        embed_partial<T, VEC, 1>
            <<<(unsigned)((n1 + WAVES - 1) / WAVES), BLOCK, 0, s>>>(
                ws.keys[at], ws.pos[at], (const T *)dout, nullptr, ws.part1,
                N, (unsigned)V, H, slices);
    const long long n2 = N / (CHUNK * CHUNK) * slices;
    if (n2)
        embed_partial<T, VEC, 2>
            <<<(unsigned)((n2 + WAVES - 1) / WAVES), BLOCK, 0, s>>>(
                ws.keys[at], ws.pos[at], nullptr, ws.part1, ws.part2, N,
                (unsigned)V, H, slices);
    const long long units = V * slices;
    long long blocks = (units + WAVES - 1) / WAVES;
    if (blocks > 1 << 20) blocks = 1 << 20;
    embed_rows<T, W, VEC><<<(unsigned)blocks, BLOCK, 0, s>>>(
        ws.spans, ws.pos[at], (const T *)dout, ws.part1, ws.part2, (W *)dw,
        units, H, slices, scale);
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t sums_vec(const Workspace &ws, int at, const void *dout, void *dw,
                    long long N, long long V, int H, float scale,
                    hipStream_t s)
{
    if (H % 8 == 0 && aligned16(dout) && aligned16(dw))
        return sums<T, W, true>(ws, at, dout, dw, N, V, H, scale, s);
    return sums<T, W, false>(ws, at, dout, dw, N, V, H, scale, s);
}

// the limits that the kernels' 32-bit counts and grids rest on
bool fits(long long N, long long V, int H)
{
    return N >= 0 && N < 1ll << 30 && V > 0 && V < 1ll << 30 && H > 0 &&
           H <= 1 << 20 &&
           (N / CHUNK + 1) * ((H + COLS - 1) / COLS) < 1ll << 30;
}

}  // namespace

extern "C" {

size_t kf_embed_ws(long long N, long long V, int H)
{
    return Workspace(nullptr, N, V, H).bytes;
}

// dtype codes: 0 f32, 1 bf16, 2 f16
hipError_t kf_embed_fwd(const void *ids, int wide, const void *weight,
                        long long ldw, int wtype, void *out, int otype,
                        long long N, long long V, int H, float scale,
                        void *stream)
{
    if (!fits(N, V, H)) return hipErrorInvalidValue;
    if (N == 0) return hipSuccess;
    hipStream_t s = (hipStream_t)stream;
#define CASE(WT, WI, OT, OI)                                                \
    if (wtype == WI && otype == OI)                                         \
    return fwd<WT, OT>(ids, wide, weight, ldw, out, N, V, H, scale, s)
    CASE(float, 0, float, 0);
    CASE(float, 0, __bf16, 1);
    CASE(float, 0, _Float16, 2);
    CASE(__bf16, 1, float, 0);
    CASE(__bf16, 1, __bf16, 1);
    CASE(_Float16, 2, float, 0);
    CASE(_Float16, 2, _Float16, 2);
#undef CASE
    return hipErrorInvalidValue;
}

hipError_t kf_embed_bwd(const void *ids, int wide, const void *dout,
                        int otype, void *dw, int wtype, long long N,
                        long long V, int H, long long padding, float scale,
                        void *work, void *stream)
{
    if (!fits(N, V, H)) return hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    const Workspace ws((char *)work, N, V, H);
    const int nb = (int)(N / SORT_TILE + 1);
    int bits = 1;
    while (V >> bits) ++bits;  // keys run to V itself
    const int passes = (bits + MAX_BITS - 1) / MAX_BITS;
    const int per = (bits + passes - 1) / passes;
    for (int p = 0; p < passes; ++p) {
        const int to = p % 2, from = 1 - to;
        if (p == 0) {
            sort_hist<true><<<nb, BLOCK, 0, s>>>(ids, wide, N, V, padding, 0,
                                                 per, ws.hist, nb, ws.spans);
        } else {
            sort_hist<false><<<nb, BLOCK, 0, s>>>(ws.keys[from], 0, N, V,
                                                  padding, p * per, per,
                                                  ws.hist, nb, ws.spans);
        }
        sort_scan<<<1, 1024, 0, s>>>(ws.hist, nb << per);
        if (p == 0)
            sort_scatter<true><<<nb, BLOCK, 0, s>>>(
                ids, wide, nullptr, N, V, padding, 0, per, ws.hist, nb,
                ws.keys[to], ws.pos[to]);
        else
            sort_scatter<false><<<nb, BLOCK, 0, s>>>(
                ws.keys[from], 0, ws.pos[from], N, V, padding, p * per, per,
                ws.hist, nb, ws.keys[to], ws.pos[to]);
    }
    const int at = (passes - 1) % 2;
    if (N)
        token_bounds<<<(unsigned)((N + BLOCK - 1) / BLOCK), BLOCK, 0, s>>>(
            ws.keys[at], N, (unsigned)V, ws.spans);
#define CASE(WT, WI, OT, OI)                                                \
    if (wtype == WI && otype == OI)                                         \
    return sums_vec<OT, WT>(ws, at, dout, dw, N, V, H, scale, s)
    CASE(float, 0, float, 0);
    CASE(float, 0, __bf16, 1);
    CASE(float, 0, _Float16, 2);
    CASE(__bf16, 1, float, 0);
    CASE(__bf16, 1, __bf16, 1);
    CASE(_Float16, 2, float, 0);
    CASE(_Float16, 2, _Float16, 2);
#undef CASE
    return hipErrorInvalidValue;
}

}  // extern "C"
