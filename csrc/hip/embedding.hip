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
constexpr int WAVES = BLOCK / WAVE;
constexpr int MAX_BITS = 8;               // digit bits of one pass
constexpr int MAX_DIGITS = 1 << MAX_BITS;
constexpr int SORT_TILE = 1024;           // keys a block ranks in one pass
constexpr int SORT_ROUNDS = SORT_TILE / BLOCK;
constexpr int SELF_SCAN = 128; // blocks up to which each finds its own places
constexpr int SMALL = 8192;    // keys up to which one block sorts them all
constexpr int SMALL_BLOCK = 1024;
constexpr int CHUNK = 32;                 // rows that one partial sum joins
constexpr int COLS = WAVE * 8;            // columns that one wave sums
constexpr int TWO_LEVELS = 16384;  // ids from which partial sums are joined

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
// 16-byte aligned), so that neighbours always touch neighbouring bytes,
// several pieces at a time: the ids' loads go out together, and then the
// rows'. Bound by memory: 65536 ids, 1024 columns of bf16, are 268 MB with
// every row read, 42 us (6.4 TB/s, rows of frequent tokens from the caches).
template <typename W, typename O, bool VEC>
__global__ __launch_bounds__(BLOCK) void embed_fwd(
    const void *__restrict__ ids, int wide, const W *__restrict__ weight,
    long long ldw, O *__restrict__ out, long long N, long long V, int H,
    int rows, float scale)
{
    constexpr int U = VEC ? 4 : 8, E = VEC ? 8 : 1;
    const int per = H / E;
    for (long long n0 = (long long)blockIdx.x * rows; n0 < N;
         n0 += (long long)gridDim.x * rows) {
        const int here = (int)(N - n0 < rows ? N - n0 : rows);
        const int all = here * per;
        for (int i0 = threadIdx.x; i0 < all; i0 += U * BLOCK) {
            int r[U], c[U];
            bool ok[U];
            long long id[U];
            float f[U][E];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                int i = i0 + u * BLOCK;
                i = i < all ? i : all - 1;
                r[u] = i / per;
                c[u] = (i - r[u] * per) * E;
                id[u] = wide ? ((const long long *)ids)[n0 + r[u]]
                             : (long long)((const int *)ids)[n0 + r[u]];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ok[u] = id[u] >= 0 && id[u] < V;
                const W *p = weight + (ok[u] ? id[u] : 0) * ldw + c[u];
                if (VEC)
                    ld8<W>(f[u], p);
                else
                    f[u][0] = (float)*p;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + u * BLOCK >= all) break;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    f[u][j] = ok[u] ? f[u][j] * scale : __builtin_nanf("");
                O *to = out + (n0 + r[u]) * H + c[u];
                if (VEC)
                    st8<O>(to, f[u]);
                else
                    *to = (O)f[u][0];
            }
        }
    }
}

// ---- stable radix sort of (token, position), least digit first ----

// No token has rows until their bounds are found.
__device__ inline void clear_spans(int *spans, long long V, long long at,
                                   long long step)
{
    for (long long i = at; i < 2 * V; i += step) spans[i] = 0;
}

// Rank of each lane's digit among those of its wave that came before, in
// the wave's own counters.
__device__ inline unsigned wave_rank(unsigned d, bool in, int bits, int lane,
                                     unsigned *cnt)
{
    unsigned long long same = __ballot(in);  // lanes with the same digit
    for (int b = 0; b < bits; ++b) {
        const unsigned long long one = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? one : ~one;
    }
    const unsigned before =
        __builtin_popcountll(same & ((1ull << lane) - 1));
    const unsigned rank = *(volatile unsigned *)&cnt[d] + before;
    __builtin_amdgcn_wave_barrier();
    if (in && before == 0)
        *(volatile unsigned *)&cnt[d] = rank + __builtin_popcountll(same);
    __builtin_amdgcn_wave_barrier();
    return rank;
}

// Exclusive prefix sum over the N threads of a block, and the total.
template <int N>
__device__ inline unsigned block_scan(unsigned v, unsigned *wsum,
                                      unsigned &total)
{
    const int lane = threadIdx.x % WAVE, w = threadIdx.x / WAVE;
    unsigned inc = v;
    for (int off = 1; off < WAVE; off <<= 1) {
        const unsigned t = __shfl_up(inc, off);
        if (lane >= off) inc += t;
    }
    if (lane == WAVE - 1) wsum[w] = inc;
    __syncthreads();
    unsigned before = 0;
    total = 0;
    for (int k = 0; k < N / WAVE; ++k) {
        if (k < w) before += wsum[k];
        total += wsum[k];
    }
    __syncthreads();
    return before + inc - v;
}

// Few ids: block 0 sorts them all, keys and places in registers, one trip
// through LDS for each digit; the other blocks clear the spans. 4096 ids of
// 30522 tokens take 14 us in one launch (the four launches below 21 us for
// 14315 ids).
__global__ __launch_bounds__(SMALL_BLOCK) void sort_small(
    const void *__restrict__ ids, int wide, int N, long long V,
    long long padding, int passes, int per, unsigned *__restrict__ keys,
    unsigned *__restrict__ pos, int *__restrict__ spans)
{
    constexpr int ITEMS = SMALL / SMALL_BLOCK, NW = SMALL_BLOCK / WAVE;
    __shared__ unsigned lkey[SMALL];
    __shared__ unsigned short lpos[SMALL];
    __shared__ unsigned cnt[NW][MAX_DIGITS];
    __shared__ unsigned wsum[NW];
    if (blockIdx.x) {
        clear_spans(spans, V,
                    (long long)(blockIdx.x - 1) * SMALL_BLOCK + threadIdx.x,
                    (long long)(gridDim.x - 1) * SMALL_BLOCK);
        return;
    }
    const int lane = threadIdx.x % WAVE, w = threadIdx.x / WAVE;
    // a wave's keys lie together, so that wave order is key order; fewer
    // keys are fewer rounds of every wave
    const int rounds = (N + SMALL_BLOCK - 1) / SMALL_BLOCK;
    const int base = w * rounds * WAVE + lane;
    unsigned key[ITEMS], p[ITEMS], rank[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int n = base + r * WAVE;
        key[r] = r < rounds && n < N ? load_key(ids, wide, n, V, padding)
                                     : 0u;
        p[r] = n;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * per;
        const unsigned mask = (1u << per) - 1;
        for (int i = threadIdx.x; i < NW * MAX_DIGITS; i += SMALL_BLOCK)
            (&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r)
            if (r < rounds)
                rank[r] = wave_rank((key[r] >> shift) & mask,
                                    base + r * WAVE < N, per, lane, cnt[w]);
        __syncthreads();
        // places: digit by digit, and wave by wave within one
        constexpr int EACH = MAX_DIGITS * NW / SMALL_BLOCK;
        const int d = threadIdx.x * EACH / NW;
        const int w0 = threadIdx.x * EACH % NW;
        unsigned c[EACH], sum = 0, total;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            c[j] = cnt[w0 + j][d];
            sum += c[j];
        }
        unsigned at = block_scan<SMALL_BLOCK>(sum, wsum, total);
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            cnt[w0 + j][d] = at;
            at += c[j];
        }
        __syncthreads();
        const bool last = pass == passes - 1;
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            if (r < rounds && base + r * WAVE < N) {
                const unsigned to =
                    cnt[w][(key[r] >> shift) & mask] + rank[r];
                if (last) {
                    keys[to] = key[r];
                    pos[to] = p[r];
                } else {
                    lkey[to] = key[r];
                    lpos[to] = (unsigned short)p[r];
                }
            }
        }
        if (last) break;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            const int n = base + r * WAVE;
            if (r < rounds && n < N) {
                key[r] = lkey[n];
                p[r] = lpos[n];
            }
        }
    }
}

// More ids: for each digit, hist counts the digits of each tile and scatter
// ranks the keys of a tile in order and moves them; with many tiles, scan
// turns the counts (digit-major) into first places in between. FIRST reads
// the ids themselves; blocks past the last tile only clear the spans.
template <bool FIRST>
__global__ __launch_bounds__(BLOCK) void sort_hist(
    const void *__restrict__ src, int wide, long long N, long long V,
    long long padding, int shift, int bits, unsigned *__restrict__ hist,
    int nb, int *__restrict__ spans)
{
    __shared__ unsigned cnt[MAX_DIGITS];
    if (FIRST)
        clear_spans(spans, V, (long long)blockIdx.x * BLOCK + threadIdx.x,
                    (long long)gridDim.x * BLOCK);
    if ((int)blockIdx.x >= nb) return;
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * SORT_TILE + threadIdx.x;
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const long long n = base + r * BLOCK;
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
    unsigned carry = 0;
    for (int base = 0; base < n; base += 1024 * 4) {
        const int i0 = base + (int)threadIdx.x * 4;
        unsigned v[4], s = 0, all;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = i0 + j < n ? hist[i0 + j] : 0;
            s += v[j];
        }
        unsigned before = carry + block_scan<1024>(s, wsum, all);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i0 + j < n) hist[i0 + j] = before;
            before += v[j];
        }
        carry += all;
    }
}

// SCANNED: `place` holds first places; else counts, of at most SELF_SCAN
// tiles, which every block sums for itself.
template <bool FIRST, bool SCANNED>
__global__ __launch_bounds__(BLOCK) void sort_scatter(
    const void *__restrict__ src, int wide,
    const unsigned *__restrict__ src_pos, long long N, long long V,
    long long padding, int shift, int bits,
    const unsigned *__restrict__ place, int nb, unsigned *__restrict__ dst,
    unsigned *__restrict__ dst_pos)
{
    // keys of one wave lie together, so wave order is key order
    __shared__ unsigned cnt[WAVES][MAX_DIGITS];
    __shared__ unsigned wsum[WAVES];
    const int lane = threadIdx.x % WAVE, w = threadIdx.x / WAVE;
    for (int i = threadIdx.x; i < WAVES * MAX_DIGITS; i += BLOCK)
        (&cnt[0][0])[i] = 0;
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
    const int d = threadIdx.x;
    unsigned at = 0;
    if (SCANNED) {
        if (d < 1 << bits) at = place[(long long)d * nb + blockIdx.x];
    } else {
        unsigned mine = 0, all = 0, total;
        if (d < 1 << bits) {
#pragma unroll 8
            for (int i = 0; i < nb; ++i) {
                const unsigned c = place[d * nb + i];
                if (i < (int)blockIdx.x) mine += c;
                all += c;
            }
        }
        at = block_scan<BLOCK>(all, wsum, total) + mine;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r)
        rank[r] = wave_rank((key[r] >> shift) & ((1u << bits) - 1),
                            base + r * WAVE < N, bits, lane, cnt[w]);
    __syncthreads();
    if (d < 1 << bits) {
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

// ---- sums of the rows of each token ----
// A wave sums 512 columns, eight a lane, in groups of `PER` neighbours: as
// many as 16 bytes of dW hold (VEC), or one by one.
template <typename W, bool VEC>
struct Cols {
    static constexpr int PER = VEC ? 16 / (int)sizeof(W) : 1;
    static constexpr int GROUPS = 8 / PER;
    // first column of the lane's group g
    static __device__ inline int at(int c0, int lane, int g)
    {
        return c0 + (g * WAVE + lane) * PER;
    }
};

template <typename T, int PER>
struct Piece {
    static constexpr int A = PER * sizeof(T) < 16 ? PER * sizeof(T) : 16;
    typedef __attribute__((ext_vector_type(PER), aligned(A))) T type;
};
template <typename T, int PER>
__device__ inline void store_n(T *p, const float *f)
{
    typedef typename Piece<T, PER>::type V;
    V v;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = (T)f[i];
    *(V *)p = v;
}

// acc += rows of `base`, `n` of them at most U, that idx(i) numbers: all
// loads go out before the first sum.
template <typename T, typename C, int U, typename Idx>
__device__ inline void add_rows(float *acc, const T *base, int n, int c0,
                                int lane, int H, Idx idx)
{
    typedef typename Piece<T, C::PER>::type V;
    V f[U][C::GROUPS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const T *row = base + (long long)idx(u < n ? u : 0) * H;
#pragma unroll
        for (int g = 0; g < C::GROUPS; ++g) {
            // a branch around a load would wait for it; lanes past the
            // last column repeat it, and their sums are not stored
            const int c = C::at(c0, lane, g);
            f[u][g] = *(const V *)(row + (c < H ? c : H - C::PER));
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                acc[j] += (float)f[u][j / C::PER][j % C::PER];
}

// Sums of CHUNK neighbours of the sorted order that belong to one token,
// so that a frequent token's row is not one long chain of reads. Level 1
// sums rows of dout and finds where each token's places begin and end;
// level 2 sums level 1's results.
template <typename T, typename W, bool VEC, int LEVEL>
__global__ __launch_bounds__(BLOCK) void embed_partial(
    const unsigned *__restrict__ keys, const unsigned *__restrict__ pos,
    const T *__restrict__ dout, const float *__restrict__ part1,
    float *__restrict__ part, int *__restrict__ spans, long long N,
    unsigned V, int H, int slices)
{
    typedef Cols<W, VEC> C;
    constexpr int SPAN = LEVEL == 1 ? CHUNK : CHUNK * CHUNK;
    const int lane = threadIdx.x % WAVE;
    const int unit = __builtin_amdgcn_readfirstlane(
        (int)(blockIdx.x * WAVES + threadIdx.x / WAVE));
    const int chunk = unit / slices, slice = unit - chunk * slices;
    const long long i0 = (long long)chunk * SPAN;
    if (i0 >= N) return;
    if (LEVEL == 1 && slice == 0 && lane < CHUNK && i0 + lane < N) {
        const long long n = i0 + lane;
        const unsigned k = keys[n];
        if (k < V) {
            if (n == 0 || keys[n - 1] != k)
                spans[2 * (long long)k] = (int)n;
            if (n == N - 1 || keys[n + 1] != k)
                spans[2 * (long long)k + 1] = (int)n + 1;
        }
    }
    if (i0 + SPAN > N) return;
    const unsigned k = keys[i0];
    if (k >= V || keys[i0 + SPAN - 1] != k) return;
    const int c0 = slice * COLS;
    float acc[8] = {};
#pragma unroll 1
    for (int i = 0; i < CHUNK; i += 16) {
        if (LEVEL == 1)
            add_rows<T, C, 16>(acc, dout, 16, c0, lane, H,
                               [&](int u) { return pos[i0 + i + u]; });
        else
            add_rows<float, C, 16>(acc, part1, 16, c0, lane, H, [&](int u) {
                return chunk * CHUNK + i + u;
            });
    }
    float *row = part + (long long)chunk * H;
#pragma unroll
    for (int g = 0; g < C::GROUPS; ++g) {
        const int c = C::at(c0, lane, g);
        if (c < H) store_n<float, C::PER>(row + c, &acc[g * C::PER]);
    }
}

// One wave writes 512 columns of one row of dW: zeros, or the token's rows
// in their order, whole chunks (and chunks of chunks, where part2 holds
// them) by their partial sums. Bound by memory, with rows of dout read in
// the tokens' order: 65536 ids of 50000 tokens, 1024 columns of bf16, are
// 237 MB in 55 us (4.3 TB/s); the sort and the chunks before take 30 us.
template <typename T, typename W, bool VEC>
__global__ __launch_bounds__(BLOCK) void embed_rows(
    const int *__restrict__ spans, const unsigned *__restrict__ pos,
    const T *__restrict__ dout, const float *__restrict__ part1,
    const float *__restrict__ part2, W *__restrict__ dw, long long units,
    int H, int slices, float scale)
{
    typedef Cols<W, VEC> C;
    // rows on their way at once: 32 registers of them
    constexpr int U = sizeof(T) == 2 ? 8 : 4;
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
            constexpr int BIG = CHUNK * CHUNK;
            const int left = end - i;
            if (i % CHUNK || left < CHUNK) {
                // up to the next chunk, or to the end
                const int here = CHUNK - i % CHUNK;
                int n = here < left ? here : left;
                n = n < U ? n : U;
                // no more loads than twice the rows that are there
                auto row = [&](int k) { return pos[i + k]; };
                if (n > 4)
                    add_rows<T, C, U>(acc, dout, n, c0, lane, H, row);
                else if (n > 2)
                    add_rows<T, C, 4>(acc, dout, n, c0, lane, H, row);
                else if (n > 1)
                    add_rows<T, C, 2>(acc, dout, n, c0, lane, H, row);
                else
                    add_rows<T, C, 1>(acc, dout, n, c0, lane, H, row);
                i += n;
            } else if (!part2 || i % BIG || left < BIG) {
                // up to the next chunk of chunks, or to the last chunk
                int n = left / CHUNK;
                const int here = (BIG - i % BIG) / CHUNK;
                n = part2 && here < n ? here : n;
                n = n < 4 ? n : 4;
                add_rows<float, C, 4>(acc, part1, n, c0, lane, H, [&](int k) {
                    return i / CHUNK + k;
                });
                i += n * CHUNK;
            } else {
                int n = left / BIG;
                n = n < 4 ? n : 4;
                add_rows<float, C, 4>(acc, part2, n, c0, lane, H,
                                      [&](int k) { return i / BIG + k; });
                i += n * BIG;
            }
        }
        W *row = dw + (long long)v * H;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] *= scale;
#pragma unroll
        for (int g = 0; g < C::GROUPS; ++g) {
            const int c = C::at(c0, lane, g);
            if (c < H) store_n<W, C::PER>(row + c, &acc[g * C::PER]);
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
        const long long nb = (N + SORT_TILE - 1) / SORT_TILE;
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
    // one turn of a block's threads, or a row
    const int turn = (vec ? 4 : 8) * BLOCK;
    const int rows = per >= turn ? 1 : turn / per;
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
    const long long n1 = (N + CHUNK - 1) / CHUNK * slices;
    if (n1)
        embed_partial<T, W, VEC, 1>
            <<<(unsigned)((n1 + WAVES - 1) / WAVES), BLOCK, 0, s>>>(
                ws.keys[at], ws.pos[at], (const T *)dout, nullptr, ws.part1,
                ws.spans, N, (unsigned)V, H, slices);
    const float *part2 = nullptr;
    if (N >= TWO_LEVELS) {
        part2 = ws.part2;
        const long long n2 = N / (CHUNK * CHUNK) * slices;
        embed_partial<T, W, VEC, 2>
            <<<(unsigned)((n2 + WAVES - 1) / WAVES), BLOCK, 0, s>>>(
                ws.keys[at], ws.pos[at], nullptr, ws.part1, ws.part2,
                nullptr, N, (unsigned)V, H, slices);
    }
    const long long units = V * slices;
    long long blocks = (units + WAVES - 1) / WAVES;
    if (blocks > 1 << 20) blocks = 1 << 20;
    embed_rows<T, W, VEC><<<(unsigned)blocks, BLOCK, 0, s>>>(
        ws.spans, ws.pos[at], (const T *)dout, ws.part1, part2, (W *)dw,
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
           (N / CHUNK + 1) * ((H + COLS - 1) / COLS) <= 1ll << 25;
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
    const int nb = (int)((N + SORT_TILE - 1) / SORT_TILE);
    int bits = 1;
    while (V >> bits) ++bits;  // keys run to V itself
    const int passes = (bits + MAX_BITS - 1) / MAX_BITS;
    const int per = (bits + passes - 1) / passes;
    // blocks beside those that sort, to clear the spans 16 ints a thread
    const long long clear = 2 * V / (16 * BLOCK) + 1;
    int at = 0;
    if (N <= SMALL) {
        const long long n = clear * BLOCK / SMALL_BLOCK + 1;
        sort_small<<<1 + (unsigned)(n < 256 ? n : 256), SMALL_BLOCK, 0,
                     s>>>(ids, wide, (int)N, V, padding, passes, per,
                          ws.keys[0], ws.pos[0], ws.spans);
    } else {
        const bool scan = nb > SELF_SCAN;
        for (int p = 0; p < passes; ++p) {
            const int to = p % 2, from = 1 - to;
            if (p == 0) {
                const long long most = clear < 1024 ? clear : 1024;
                sort_hist<true>
                    <<<nb > most ? nb : (unsigned)most, BLOCK, 0, s>>>(
                        ids, wide, N, V, padding, 0, per, ws.hist, nb,
                        ws.spans);
            } else {
                sort_hist<false><<<nb, BLOCK, 0, s>>>(
                    ws.keys[from], 0, N, V, padding, p * per, per, ws.hist,
                    nb, nullptr);
            }
            if (scan) sort_scan<<<1, 1024, 0, s>>>(ws.hist, nb << per);
            auto scatter = p == 0 ? (scan ? sort_scatter<true, true>
                                          : sort_scatter<true, false>)
                                  : (scan ? sort_scatter<false, true>
                                          : sort_scatter<false, false>);
            scatter<<<nb, BLOCK, 0, s>>>(
                p == 0 ? ids : ws.keys[from], wide, ws.pos[from], N, V,
                padding, p * per, per, ws.hist, nb, ws.keys[to], ws.pos[to]);
            at = to;
        }
    }
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
