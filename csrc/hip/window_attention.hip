// Attention with a sliding window and first tokens that stay visible,
// forward and backward — gfx950.
//
//   out = softmax(scale * q k^T over the visible keys) v
// A query at position p of a sequence of n keys sees key j when j < n and
// (|p - j| < window or j < sinks), and j <= p where causal. A query whose
// position is outside [0, n) sees nothing: its output and gradients are 0.
//
// The G query heads that share a key head are flattened with the queries:
// row r of a key head is query r / G, head r % G. Positions grow with r,
// so a block of rows is a block of neighbouring queries, and one pass over
// the keys serves the whole group.
//
// All three kernels keep one operand of 32 columns per wave in registers
// and stream tiles of the others through LDS. Scores are computed as
// S^T = K Q^T (forward, dq; a column is a query) or S = Q K^T (dk, dv; a
// column is a key), with mfma 32x32x16: lane l holds column l % 32 and,
// in accumulator r, row 8 (r / 4) + 4 (l / 32) + r % 4. The second
// product contracts over those rows, and any order of the contracted
// index will do as long as both operands share it: eight accumulators,
// rounded to 16 bits, are the B operand as they are, and the A operand is
// read from the same LDS tile by the transposing 64-bit read with the rows
// in that order. No probability passes through LDS or between lanes.
//
// Long rows are bound by the matrix pipe, which the softmax's vector work
// beside it keeps from its full rate: 2 x 8192 tokens, 16 heads, no mask,
// forward 1096 us at 128 columns (1003 TFLOP/s) and 615 us at 64 (894), dq
// 1579 us (1044) and 911 us (905), dk and dv 2239 us (982) and 1235 us
// (890). Few rows over many keys are bound by the reads of k and v.
//
// The backward computes the scores twice, once for dq and once for dk and
// dv, instead of adding dq with atomics: every output is written once by
// one block in a fixed order, so results repeat bit by bit.
//
// Probabilities and their gradients are rounded to the inputs' 16 bits as
// operands of the second product (their relative error of half a step is
// that of the inputs themselves); scores, softmax statistics, sums and
// accumulators are f32.
#include <climits>

#include "vec.hpp"

using namespace kfv;

namespace {

constexpr int TILE = 64;  // rows of a streamed tile
constexpr int KT = TILE;

struct Args {
    const void *q, *k, *v, *dout, *o, *orest;
    void *out, *rest, *dq, *dk, *dv;
    float *lse, *delta;  // [B][Hk][S * G]; lse in powers of two
    long long qb, qs, qh, kb, ks, kh, vb, vs, vh, gb, gs, gh;
    int B, S, T, Hk, G, D;
    int window, sinks, causal;
    const int *lengths, *starts;
    float scale, c;  // c = scale * log2(e)
    int keys;        // of a block of dk and dv
    int blocks;      // row blocks (or key blocks) of a key head
    int splits;
    float *part_o, *part_ml;     // forward and dq, split over keys
    float *part_k, *part_v;      // dk, dv, split over rows
    int sink_blocks, sink_splits, splits_rows, sink_rows;
    int even;  // G divides a tile's rows, whose offsets fit 32 bits
    int few;   // rows see few keys: delta is summed over them
};

template <typename T>
__device__ inline f32x16 mfma(s16x8 a, s16x8 b, f32x16 c);
template <>
__device__ inline f32x16 mfma<__bf16>(s16x8 a, s16x8 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
        0, 0);
}
template <>
__device__ inline f32x16 mfma<_Float16>(s16x8 a, s16x8 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
        0);
}

// Sixteen accumulators of a column as 16-bit values: rows 8 x + 0..7 of x =
// 2 i + l / 32 in to[i], one piece of 16 bytes, which the lanes of the two
// halves exchange parts for.
template <typename T>
__device__ inline void pack16(const f32x16 &x, s16x8 (&to)[2])
{
    typedef __attribute__((ext_vector_type(4))) T T4;
    typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
    typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        T4 a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = (T)x[i * 8 + j];
            b[j] = (T)x[i * 8 + 4 + j];
        }
        const u32x2 u = __builtin_bit_cast(u32x2, a);
        const u32x2 v = __builtin_bit_cast(u32x2, b);
        const auto p = __builtin_amdgcn_permlane32_swap(u[0], v[0], false,
                                                        false);
        const auto q = __builtin_amdgcn_permlane32_swap(u[1], v[1], false,
                                                        false);
        const u32x4 w = {p[0], q[0], p[1], q[1]};
        to[i] = __builtin_bit_cast(s16x8, w);
    }
}

// Stores a column's 32 x DP / 32 accumulators as its row of D values.
template <typename T, int DP>
__device__ inline void store_row(T *row, const f32x16 (&x)[DP / 32], int D,
                                 int lane)
{
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
        s16x8 y[2];
        pack16<T>(x[d], y);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = d * 32 + i * 16 + lane / 32 * 8;
            if (c < D) *(s16x8 *)(row + c) = y[i];
        }
    }
}

// The same as f32.
template <int DP>
__device__ inline void store_sums(float *row, const f32x16 (&x)[DP / 32],
                                  int lane)
{
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f32x4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = x[d][e * 4 + j];
            *(f32x4 *)(row + d * 32 + e * 8 + lane / 32 * 4) = y;
        }
}

// Eight accumulators, from `at`, as a 16-bit operand.
template <typename T>
__device__ inline s16x8 pack8(const f32x16 &x, int at)
{
    typename vec8<T>::type v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)x[at + i];
    return __builtin_bit_cast(s16x8, v);
}

// LDS tile: KT rows of DP elements in chunks of 16 bytes. Tiles are filled
// by loads that go from memory to LDS without passing registers, which put
// 64 lanes' chunks one after another: rows cannot be padded apart, so the
// chunks of a row are permuted instead, c to c ^ f(row) within blocks of BS
// chunks. f takes neighbouring rows' pairs of chunks (the transposing
// read) and eight rows' single chunks (the plain one) to distinct banks.
template <int DP, int ROWS = KT>
struct Tile {
    static constexpr int CH = DP / 8;                      // chunks of a row
    static constexpr int BS = DP == 128 ? 16 : DP == 64 ? 8 : 4;
    __align__(1024) short x[ROWS * DP];

    static __device__ inline int f(int row)
    {
        if (BS == 4) return (row >> 1 & 1) << 1 | (row >> 2 & 1);
        return (row & 3) << 1 | (row >> 2 & 1) | (BS == 16 ? row & 8 : 0);
    }
    // byte of chunk `c` of `row`
    static __device__ inline int at(int row, int c)
    {
        return row * DP * 2 + ((c & -BS) + ((c & (BS - 1)) ^ f(row))) * 16;
    }
};

// A operand from rows r0..r0+31 as they lie: row r0 + l % 32, elements
// 16 ks + 8 (l / 32) + 0..7. `at` is the lane's place for ks = 0, r0 = 0.
template <int DP>
__device__ inline int rows_at(int lane)
{
    return Tile<DP>::at(lane % 32, lane / 32);
}
template <int DP, int ROWS>
__device__ inline s16x8 rows_op(const Tile<DP, ROWS> &t, int at, int r0, int ks)
{
    constexpr int BS = Tile<DP>::BS;
    const int c = ks * 2;
    return *(const s16x8 *)((const char *)t.x +
                            ((at ^ (c & (BS - 1)) << 4) + (c & -BS) * 16 +
                             r0 * DP * 2));
}

// A operand of the transposed tile: row (of the operand) = element
// 32 dt + l % 32, contracted index = tile rows r0 + 4 (l / 32) + 0..3 and
// 8 rows on, the order in which the accumulators hold them.
template <int DP>
__device__ inline int cols_at(int lane)
{
    const int i = lane % 16;
    return Tile<DP>::at(lane / 32 * 4 + i / 4,
                        lane / 16 % 2 * 2 + i % 4 / 2) +
           i % 2 * 8;
}
template <int DP, int ROWS>
__device__ inline s16x8 cols_op(const Tile<DP, ROWS> &t, int at, int r0, int dt)
{
    constexpr int BS = Tile<DP>::BS;
    const int c = dt * 4;
    const char *p = (const char *)t.x + r0 * DP * 2 + (c & -BS) * 16;
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4 *)(p + (at ^ (c & (BS - 1)) << 4)));
    // eight rows on; f has their bit where BS is 16
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4 *)(p + 8 * DP * 2 +
                 (at ^ ((c ^ (BS == 16 ? 8 : 0)) & (BS - 1)) << 4)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Loads on their way into LDS are done, for this wave's part.
__device__ inline void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Sends 16 bytes of each lane to 1 KiB of LDS from `to` (the same for all
// lanes).
__device__ inline void send16(const void *from, void *to)
{
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void *)from,
        (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

// A lane's share of a tile that NW waves fill: which row and column its
// v-th 16 bytes hold.
template <int DP, int NW, int ROWS = KT>
struct Share {
    static constexpr int CH = Tile<DP>::CH, BS = Tile<DP>::BS;
    static constexpr int N = ROWS * CH / WAVE / NW;
    static __device__ inline int row(int v, int wid, int lane)
    {
        return ((v * NW + wid) * WAVE + lane) / CH;
    }
    static __device__ inline int col(int v, int wid, int lane, int D)
    {
        const int n = (v * NW + wid) * WAVE + lane, x = n % CH;
        const int c = (x & -BS) + ((x & (BS - 1)) ^ Tile<DP>::f(n / CH));
        return c * 8 < D ? c * 8 : 0;
    }
};

// Sends rows of a matrix to a tile; at(v) is the address of the lane's v-th
// piece. Rows past the last one and columns past D repeat others, which
// hold nothing that could not stand there: their scores are masked, their
// weights are zeros, and their columns meet zeros or are not written.
template <int DP, int NW, int U, int ROWS, typename At>
__device__ inline void send_tile(Tile<DP, ROWS> &t, int wid, At at)
{
#pragma unroll U
    for (int v = 0; v < Share<DP, NW, ROWS>::N; ++v)
        send16(at(v), (char *)t.x + (v * NW + wid) * WAVE * 16);
}

// Byte offsets of a lane's pieces of a tile from its first row. Where the
// waves' loads take whole rows, the v-th piece lies `step` bytes (the same
// for all lanes) after the one before.
template <int DP, int NW, int ROWS = KT>
struct Offsets {
    typedef Share<DP, NW, ROWS> S;
    static constexpr bool WHOLE = NW * WAVE % S::CH == 0 &&
                                  NW * WAVE / S::CH % Tile<DP>::BS == 0;
    static constexpr int EACH = NW * WAVE / S::CH;  // rows of one v, if WHOLE
    unsigned off[WHOLE ? 1 : S::N];
    // row_off(row): elements of a row from the tile's first
    template <typename F>
    __device__ void set(int wid, int lane, int D, F row_off)
    {
#pragma unroll
        for (int v = 0; v < (WHOLE ? 1 : S::N); ++v)
            off[v] = 2u * (row_off(S::row(v, wid, lane)) +
                           S::col(v, wid, lane, D));
    }
    // `step`: elements from a row to the one EACH further
    __device__ void send(Tile<DP, ROWS> &t, const short *from, long long step,
                         int wid) const
    {
        send_tile<DP, NW, 16>(t, wid, [&](int v) {
            return WHOLE ? (const char *)(from + v * step) + off[0]
                         : (const char *)from + off[WHOLE ? 0 : v];
        });
    }
};

// Keys and values: rows j0.. of a [T][D] matrix. Whole tiles take the
// lane's offsets, which are the same for all of them, on a base that is
// the same for all lanes; the last tile of a sequence stops at its end.
template <int DP, int NW, int ROWS = KT>
struct KeyShare {
    typedef Share<DP, NW, ROWS> S;
    Offsets<DP, NW, ROWS> o;
    __device__ KeyShare(long long stride, int wid, int lane, int D)
    {
        o.set(wid, lane, D,
              [&](int row) { return (unsigned)row * (unsigned)stride; });
    }
    __device__ void send(Tile<DP, ROWS> &t, const short *base, long long stride,
                         int j0, int end, int wid, int lane, int D) const
    {
        if (j0 + ROWS <= end) {
            o.send(t, base + j0 * stride, Offsets<DP, NW, ROWS>::EACH * stride,
                   wid);
        } else {
            send_tile<DP, NW, 1>(t, wid, [&](int v) {
                int j = j0 + S::row(v, wid, lane);
                j = j < end ? j : end - 1;
                return base + j * stride +
                       S::col(v, wid, lane, D);
            });
        }
    }
};

// The value of the lane 32 lanes away.
__device__ inline float other_half(float x)
{
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, threadIdx.x & 32 ? r[0] : r[1]);
}

struct Seq {
    int n;      // keys
    int start;  // position of query 0
};

__device__ inline Seq sequence(const Args &a, int b)
{
    Seq s;
    s.n = a.T;
    s.start = a.T - a.S;
    if (a.lengths) {
        const int n = a.lengths[b];
        s.n = n < 0 ? 0 : n > a.T ? a.T : n;
    }
    if (a.starts) {
        const int p = a.starts[b];
        const int most = 1 << 30;
        s.start = p < -most ? -most : p > most ? most : p;
    }
    return s;
}

// What one query sees: keys [lo, hi] and [0, first).
struct View {
    int lo, hi, first;
    __device__ bool sees(int j) const
    {
        return (j >= lo && j <= hi) || j < first;
    }
};

__device__ inline View view_of(const Args &a, const Seq &s, int p)
{
    View v = {0, -1, 0};
    if (p >= 0 && p < s.n) {
        const int last = a.causal ? p : s.n - 1;
        v.lo = p - a.window + 1;
        v.hi = a.causal || a.window > last - p ? last : p + a.window - 1;
        v.first = a.sinks < last + 1 ? a.sinks : last + 1;
    }
    return v;
}

// Tiles of keys that rows at positions p0..p1 (inside the sequence) see:
// `head` tiles from key 0, then those from tile `from` up to `to`.
struct Tiles {
    int head, from, to;
    __device__ int count() const { return head + to - from; }
    __device__ int at(int i) const { return i < head ? i : from + i - head; }
};

template <int ROWS>
__device__ inline Tiles tiles_of(const Args &a, const Seq &s, int p0, int p1)
{
    Tiles t = {0, 0, 0};
    if (p0 < 0) p0 = 0;
    if (p1 > s.n - 1) p1 = s.n - 1;
    if (p0 > p1) return t;
    const View x = view_of(a, s, p0), y = view_of(a, s, p1);
    const int lo = x.lo < 0 ? 0 : x.lo;
    int hi = y.hi + 1;
    if (y.first > hi) hi = y.first;
    t.from = lo / ROWS;
    t.to = (hi + ROWS - 1) / ROWS;
    const int sinks = (y.first + ROWS - 1) / ROWS;
    t.head = sinks < t.from ? sinks : t.from;
    return t;
}

// Whether keys k0..k1 are all seen (2), partly (1) or not at all (0) by
// all queries of positions p0..p1.
__device__ inline int seen(const Args &a, const Seq &s, int p0, int p1,
                           int k0, int k1)
{
    if (p0 < 0) p0 = 0;
    if (p1 > s.n - 1) p1 = s.n - 1;
    if (p0 > p1 || k0 >= s.n) return 0;
    const View x = view_of(a, s, p0), y = view_of(a, s, p1);
    // the union of the windows is [x.lo, y.hi], their common part
    // [y.lo, x.hi]; first tokens grow with p where causal
    if (k0 >= y.first && (k0 > y.hi || k1 < x.lo)) return 0;
    if ((k0 >= y.lo && k1 <= x.hi) || k1 < x.first) return 2;
    return 1;
}

// Work is handed out head by head for each block of rows or keys, the
// blocks with most to do first: causal blocks that see much start before
// those that see little, and blocks that share a CU are of all sizes.
// Where the heads are a multiple of eight, a head stays on one XCD, since
// neighbouring workgroups go to neighbouring XCDs.

// ---- forward ----
// A wave owns 32 rows. SPLIT: the block takes one of `splits` parts of the
// row block's tiles and writes the sums as they are, for attn_join.
template <typename T, int DP, int NW, bool SPLIT>
__global__ __launch_bounds__(NW *WAVE, 2) void attn_fwd(const Args a)
{
    // One wave takes half the keys at a time, so that a CU holds four such
    // blocks at 128 columns: 16 sequences of 5 to 16 thousand keys, 32/8
    // heads, 131 us (5.3 TB/s) against 142 us.
    constexpr int KT = NW < 4 ? 32 : TILE;
    typedef Tile<DP, KT> Tile;
    __shared__ Tile kt0, kt1, vt0, vt1;
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int heads = a.B * a.Hk;
    int unit = blockIdx.x, split = 0;
    if (SPLIT) {
        unit /= a.splits;
        split = blockIdx.x - unit * a.splits;
    }
    const int blk = a.blocks - 1 - unit / heads;
    const int bh = unit % heads;
    const int b = bh / a.Hk, h = bh - b * a.Hk;
    const int SG = a.S * a.G;
    const Seq s = sequence(a, b);

    const int r0 = blk * NW * 32, w0 = r0 + wid * 32;
    const int rlast = r0 + NW * 32 < SG ? r0 + NW * 32 - 1 : SG - 1;
    const int wlast = w0 + 31 < SG ? w0 + 31 : SG - 1;
    const int r = w0 + lane % 32, qi = r / a.G, g = r - qi * a.G;
    const int p = s.start + qi;
    const View view =
        r < SG ? view_of(a, s, p) : View{0, -1, 0};
    const bool live = r < SG && p >= 0 && p < s.n;
    // positions of this wave's rows; none where it has no rows
    const int wp0 = s.start + w0 / a.G;
    const int wp1 = w0 < SG ? s.start + wlast / a.G : INT_MIN / 2;

    // loads are not branched around, which would wait for each: lanes
    // without a row, or past the last column, read others and drop them
    s16x8 qop[DP / 16];
    {
        const int rr = r < SG ? r : SG - 1, i = rr / a.G, gg = rr - i * a.G;
        const short *row = (const short *)a.q + b * a.qb + i * a.qs +
                           (long long)(h * a.G + gg) * a.qh;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const int d = i * 16 + lane / 32 * 8;
            qop[i] = *(const s16x8 *)(row + (d < a.D ? d : 0));
        }
    }

    const Tiles tl =
        tiles_of<KT>(a, s, s.start + r0 / a.G, s.start + rlast / a.G);
    int i = 0, end = tl.count();
    if (SPLIT) {
        const int n = end;
        i = (int)((long long)n * split / a.splits);
        end = (int)((long long)n * (split + 1) / a.splits);
    }
    const short *kbase = (const short *)a.k + b * a.kb + h * a.kh;
    const short *vbase = (const short *)a.v + b * a.vb + h * a.vh;

    f32x16 o[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
    float m = -__builtin_inff(), l = 0.f;

    int rat = rows_at<DP>(lane), cat = cols_at<DP>(lane);
    const KeyShare<DP, NW, KT> kshare(a.ks, wid, lane, a.D),
        vshare(a.vs, wid, lane, a.D);
    // Step u computes the scores of tile u and, in the same run of
    // instructions, the weights and products of tile u - 1, so that the
    // matrix pipe and the vector pipe both have work: 2 x 16 heads of 128,
    // 8192 tokens, 891 TFLOP/s against 847 with one tile after another. It
    // needs keys u and values u - 1 in LDS, and sends keys u + 1 and values
    // u on their way.
    auto score = [&](const Tile &kt, f32x16(&x)[KT / 32]) {
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
            x[t] = f32x16{};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d)
                x[t] = mfma<T>(rows_op<DP>(kt, rat, t * 32, d), qop[d],
                               x[t]);
        }
    };
    auto weigh = [&](const Tile &vt, f32x16(&x)[KT / 32]) {
        const float base = m == -__builtin_inff() ? 0.f : m * a.c;
        float sum[4] = {};
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
#pragma unroll
            for (int e = t % 2 * 8; e < t % 2 * 8 + 8; ++e) {
                f32x16 &y = x[t / 2];
                y[e] = __builtin_amdgcn_exp2f(y[e] * a.c - base);
                sum[e % 4] += y[e];
            }
            const s16x8 pop = pack8<T>(x[t / 2], t % 2 * 8);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
                o[d] = mfma<T>(cols_op<DP>(vt, cat, t * 16, d), pop, o[d]);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };
    // Hides what the mask hides of tile k0, and keeps m.
    auto settle = [&](int k0, f32x16(&x)[KT / 32]) {
        if (seen(a, s, wp0, wp1, k0, k0 + KT - 1) != 2) {
#pragma unroll
            for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = k0 + t * 32 + e / 4 * 8 + lane / 32 * 4 +
                                  e % 4;
                    if (!view.sees(j)) x[t][e] = -__builtin_inff();
                }
        }
        float top = x[0][0];
#pragma unroll
        for (int t = 0; t < KT / 32; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, x[t][e]);
        top = fmaxf(top, other_half(top));
        // m, which all weights are taken against, follows the maximum only
        // when that is 2^8 over it: weights up to 2^8 keep the relative
        // precision of the 16 bits they are rounded to, and the sums so
        // far are seldom scaled
        if (__any((top - m) * a.c > 8.f)) {
            const float mn = fmaxf(m, top);
            // a row that has seen nothing yet keeps zeros
            const float alpha = __builtin_amdgcn_exp2f(
                mn == -__builtin_inff() ? 0.f : (m - mn) * a.c);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
        }
    };
    // A tile that this wave sees nothing of, of those that its block sees,
    // is computed and masked as any other.
    auto ready = [&](Tile &kn, Tile &vn) {
        landed();
        __syncthreads();
        if (i + 1 < end)
            kshare.send(kn, kbase, a.ks, tl.at(i + 1) * KT, s.n, wid, lane,
                        a.D);
        if (i < end)
            vshare.send(vn, vbase, a.vs, tl.at(i) * KT, s.n, wid, lane, a.D);
    };
    auto step = [&](const Tile &kt, const Tile &vt, Tile &kn,
                    Tile &vn, f32x16(&xp)[KT / 32],
                    f32x16(&x)[KT / 32]) {
        ready(kn, vn);
        // the places that follow from these two are worked out again: kept,
        // they would take the registers of half a tile's scores
        asm volatile("" : "+v"(rat), "+v"(cat));
        // before waves that settle: 881 -> 913 TFLOP/s at 64 columns
        __builtin_amdgcn_s_setprio(1);
        score(kt, x);
        weigh(vt, xp);
        __builtin_amdgcn_s_setprio(0);
        settle(tl.at(i) * KT, x);
        ++i;
    };
    if (i < end) {
        f32x16 xa[KT / 32], xb[KT / 32];
        kshare.send(kt0, kbase, a.ks, tl.at(i) * KT, s.n, wid, lane, a.D);
        // the first tile is on its way before q is waited for
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
            if (!live || d * 16 + lane / 32 * 8 >= a.D) qop[d] = s16x8{};
        ready(kt1, vt0);
        score(kt0, xa);
        settle(tl.at(i) * KT, xa);
        ++i;
        // two buffers by name, so that reads of one are known not to touch
        // what is on its way into the other
        while (i + 1 < end) {
            step(kt1, vt0, kt0, vt1, xa, xb);
            step(kt0, vt1, kt1, vt0, xb, xa);
        }
        if (i < end) {
            step(kt1, vt0, kt0, vt1, xa, xb);
            ready(kt1, vt0);
            weigh(vt1, xb);
        } else {
            ready(kt0, vt1);
            weigh(vt0, xa);
        }
    }
    l += other_half(l);
    if (!live) {  // a tile that its neighbours see whole is not masked
        m = -__builtin_inff();
        l = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
    }
    const long long row = (long long)bh * SG + r;
    if (SPLIT) {
        if (r >= SG) return;
        // rows of a head in order, parts of a row together
        store_sums<DP>(a.part_o + (row * a.splits + split) * DP, o, lane);
        if (lane < 32) {
            float *ml = a.part_ml + (row * a.splits + split) * 2;
            ml[0] = m * a.c;
            ml[1] = l;
        }
        return;
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= inv;
    // lanes without a row take part in the exchanges, and write nothing
    const int D = r < SG ? a.D : 0;
    const long long at =
        (((long long)b * a.S + qi) * a.Hk * a.G + h * a.G + g) * a.D;
    store_row<T, DP>((T *)a.out + at, o, D, lane);
    if (a.rest) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] -= (float)(T)o[d][e];
        store_row<T, DP>((T *)a.rest + at, o, D, lane);
    }
    if (r >= SG) return;
    // a row that sees nothing has no weight anywhere: exp2(s - inf) = 0
    if (a.lse && lane < 32)
        a.lse[row] = l == 0.f ? __builtin_inff() : m * a.c + log2f(l);
}

// Joins the parts of a row where they are few: four columns a thread.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_few(const Args a)
{
    constexpr int PER = DP / 4;
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = e / PER;
    const int c = (int)(e - row * PER) * 4;
    if (row >= (long long)a.B * a.Hk * a.S * a.G) return;
    const float *ml = a.part_ml + row * a.splits * 2;
    float m = -__builtin_inff();
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) m = fmaxf(m, ml[2 * i]);
    const float base = m == -__builtin_inff() ? 0.f : m;
    float l = 0.f;
    f32x4 x = {};
    const float *po = a.part_o + row * a.splits * DP + c;
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) {
        const float w = __builtin_amdgcn_exp2f(ml[2 * i] - base);
        l += w * ml[2 * i + 1];
        x += w * *(const f32x4 *)(po + (long long)i * DP);
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    const long long bh = row / (a.S * a.G);
    const int r = (int)(row - bh * (a.S * a.G)), qi = r / a.G;
    const int g = r - qi * a.G;
    const int b = (int)(bh / a.Hk), h = (int)(bh - (long long)b * a.Hk);
    const long long at =
        (((long long)b * a.S + qi) * a.Hk * a.G + h * a.G + g) * a.D + c;
    if (c < a.D) {
        typedef __attribute__((ext_vector_type(4))) T T4;
        T4 y, z;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float f = x[j] * inv;
            y[j] = (T)f;
            z[j] = (T)(f - (float)y[j]);
        }
        *(T4 *)((T *)a.out + at) = y;
        if (a.rest) *(T4 *)((T *)a.rest + at) = z;
    }
    if (a.lse && c == 0)
        a.lse[row] = l == 0.f ? __builtin_inff() : base + log2f(l);
}

// Joins the parts of a row where they are many, one block a row: each wave
// a quarter of them in order, against the quarter's own maximum, then the
// quarters in order.
template <typename T>
__global__ __launch_bounds__(256) void attn_join(const Args a, int DP)
{
    __shared__ float mq[4], lq[4], oq[4][128];
    const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
    const long long row = blockIdx.x;
    const float *ml = a.part_ml + row * a.splits * 2;
    const int p0 = (int)((long long)a.splits * wid / 4);
    const int p1 = (int)((long long)a.splits * (wid + 1) / 4);
    float m = -__builtin_inff();
    for (int i = p0 + lane; i < p1; i += WAVE) m = fmaxf(m, ml[2 * i]);
    for (int off = WAVE / 2; off > 0; off >>= 1)
        m = fmaxf(m, __shfl_xor(m, off));
    float base = m == -__builtin_inff() ? 0.f : m;
    float l = 0.f, o[2] = {};
    // columns past DP repeat the last one and are not written
    const int c0 = lane < DP ? lane : DP - 1;
    const int c1 = lane + 64 < DP ? lane + 64 : DP - 1;
    const float *po = a.part_o + row * a.splits * DP;
#pragma unroll 8
    for (int i = p0; i < p1; ++i) {
        const float w = __builtin_amdgcn_exp2f(ml[2 * i] - base);
        l += w * ml[2 * i + 1];
        o[0] += w * po[(long long)i * DP + c0];
        o[1] += w * po[(long long)i * DP + c1];
    }
    if (lane == 0) {
        mq[wid] = m;
        lq[wid] = l;
    }
    oq[wid][lane] = o[0];
    oq[wid][lane + 64] = o[1];
    __syncthreads();
    m = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
    base = m == -__builtin_inff() ? 0.f : m;
    const int c = threadIdx.x % 128;
    float x = 0.f;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float w = __builtin_amdgcn_exp2f(mq[i] - base);
        l += w * lq[i];
        x += w * oq[i][c];
    }
    const float f = l > 0.f ? x / l : l == 0.f ? 0.f : l;
    const long long bh = row / (a.S * a.G);
    const int r = (int)(row - bh * (a.S * a.G)), qi = r / a.G;
    const int g = r - qi * a.G;
    const int b = (int)(bh / a.Hk), h = (int)(bh - (long long)b * a.Hk);
    const long long at =
        (((long long)b * a.S + qi) * a.Hk * a.G + h * a.G + g) * a.D + c;
    if (threadIdx.x < 128 && c < a.D) {
        ((T *)a.out)[at] = (T)f;
        if (a.rest) ((T *)a.rest)[at] = (T)(f - (float)(T)f);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[row] = l == 0.f ? __builtin_inff() : base + log2f(l);
}

// ---- backward: dq, and delta = sum(dout * out) of each row ----
// The output is read with what its rounding took off (`rest`, which the
// forward keeps): delta is subtracted from every gradient of a weight, and
// the rounding of 16 bits in it alone would add a tenth to the error of dq
// and dk (at 2048 causal tokens 0.0025 of their norm, 0.0024 with it, where
// the rounding of dq itself is 0.0017). The output also carries the rounding
// of the weights that it was summed with, which cancels over many keys and
// not over few. Where rows see no more than FEW_KEYS, delta is summed over them
// instead, weight times gradient of the weight in f32, in a pass of its own:
// dq and dk are off by 0.0025 of their norm instead of 0.0028 at 3 keys a
// row, 0.0024 instead of 0.0025 at 9, and a training step of 8192 tokens,
// 32/8 heads of 128, window 16, takes 293 us instead of 278.
// SPLIT: the block takes one of `splits` parts of the row block's tiles and
// writes its f32 sums, for attn_join_dq.
template <typename T, int DP, int NW, bool SPLIT>
__global__
__launch_bounds__(NW *WAVE, DP > 64 ? 2 : 3) void attn_dq(const Args a)
{
    constexpr int KT = NW < 4 ? 32 : TILE;
    typedef Tile<DP, KT> Tile;
    __shared__ Tile kt0, kt1, vt0, vt1;
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int heads = a.B * a.Hk;
    int unit = blockIdx.x, split = 0;
    if (SPLIT) {
        unit /= a.splits;
        split = blockIdx.x - unit * a.splits;
    }
    const int blk = a.blocks - 1 - unit / heads, bh = unit % heads;
    const int b = bh / a.Hk, h = bh - b * a.Hk;
    const int SG = a.S * a.G;
    const Seq s = sequence(a, b);
    const int r0 = blk * NW * 32, w0 = r0 + wid * 32;
    const int rlast = r0 + NW * 32 < SG ? r0 + NW * 32 - 1 : SG - 1;
    const int wlast = w0 + 31 < SG ? w0 + 31 : SG - 1;
    const int r = w0 + lane % 32, qi = r / a.G, g = r - qi * a.G;
    const int p = s.start + qi;
    const View view = r < SG ? view_of(a, s, p) : View{0, -1, 0};
    const bool live = r < SG && p >= 0 && p < s.n;
    const int wp0 = s.start + w0 / a.G;
    const int wp1 = w0 < SG ? s.start + wlast / a.G : INT_MIN / 2;
    const int head = h * a.G + g;
    const long long row = (long long)bh * SG + r;
    const long long orow =
        (((long long)b * a.S + qi) * a.Hk * a.G + head) * a.D;

    s16x8 qop[DP / 16], gop[DP / 16];
    typedef typename vec8<T>::type T8;
    T8 o[DP / 16], rest[DP / 16];
    {
        const int rr = r < SG ? r : SG - 1, i = rr / a.G;
        const int hh = h * a.G + rr - i * a.G;
        const short *qrow = (const short *)a.q + b * a.qb + i * a.qs +
                            (long long)hh * a.qh;
        const short *grow = (const short *)a.dout + b * a.gb + i * a.gs +
                            (long long)hh * a.gh;
        const long long at =
            (((long long)b * a.S + i) * a.Hk * a.G + hh) * a.D;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            int d = i * 16 + lane / 32 * 8;
            d = d < a.D ? d : 0;
            gop[i] = *(const s16x8 *)(grow + d);
            o[i] = *(const T8 *)((const T *)a.o + at + d);
            rest[i] = *(const T8 *)((const T *)a.orest + at + d);
            qop[i] = *(const s16x8 *)(qrow + d);
        }
    }
    const float kept = a.lse[(long long)bh * SG + (r < SG ? r : SG - 1)];

    const Tiles tl =
        tiles_of<KT>(a, s, s.start + r0 / a.G, s.start + rlast / a.G);
    int i = 0, end = tl.count();
    if (SPLIT) {
        const int n = end;
        i = (int)((long long)n * split / a.splits);
        end = (int)((long long)n * (split + 1) / a.splits);
    }
    const short *kbase = (const short *)a.k + b * a.kb + h * a.kh;
    const short *vbase = (const short *)a.v + b * a.vb + h * a.vh;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = f32x16{};

    const int rat = rows_at<DP>(lane), cat = cols_at<DP>(lane);
    const KeyShare<DP, NW, KT> kshare(a.ks, wid, lane, a.D),
        vshare(a.vs, wid, lane, a.D);
    auto send = [&](int tile, Tile &kt, Tile &vt) {
        kshare.send(kt, kbase, a.ks, tile * KT, s.n, wid, lane, a.D);
        vshare.send(vt, vbase, a.vs, tile * KT, s.n, wid, lane, a.D);
    };
    // the first tiles are on their way before the rows are waited for
    if (i < end) send(tl.at(i), kt0, vt0);
    float delta = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        if (!live || i * 16 + lane / 32 * 8 >= a.D)
            qop[i] = gop[i] = s16x8{};
        const T8 z = __builtin_bit_cast(T8, gop[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            delta += ((float)o[i][j] + (float)rest[i][j]) * (float)z[j];
    }
    delta += other_half(delta);
    const float lse = r < SG ? kept : __builtin_inff();
    if (!SPLIT && a.few) {
        delta = 0.f;
        for (int n = i; n < end; ++n) {
            const int k0 = tl.at(n) * KT;
            landed();
            __syncthreads();
            const int see = seen(a, s, wp0, wp1, k0, k0 + KT - 1);
#pragma unroll
            for (int t = 0; t < KT / 32; ++t) {
                if (see == 0) break;
                f32x16 x = {}, y = {};
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    x = mfma<T>(rows_op<DP>(kt0, rat, t * 32, d), qop[d], x);
                    y = mfma<T>(rows_op<DP>(vt0, rat, t * 32, d), gop[d], y);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = k0 + t * 32 + e / 4 * 8 + lane / 32 * 4 +
                                  e % 4;
                    const float w =
                        __builtin_amdgcn_exp2f(x[e] * a.c - lse) * y[e];
                    delta += view.sees(j) ? w : 0.f;
                }
            }
            __syncthreads();
            // the next tile, and after the last one the first again
            send(tl.at(n + 1 < end ? n + 1 : i), kt0, vt0);
        }
        delta += other_half(delta);
    }
    if (r < SG && lane < 32 && split == 0) a.delta[row] = delta;
    auto step = [&](const Tile &kt, const Tile &vt, Tile &kn,
                    Tile &vn) {
        const int k0 = tl.at(i) * KT;
        landed();
        __syncthreads();
        if (i + 1 < end) send(tl.at(i + 1), kn, vn);
        const int see = seen(a, s, wp0, wp1, k0, k0 + KT - 1);
        if (see == 0) return;
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
            f32x16 x = {}, y = {};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                x = mfma<T>(rows_op<DP>(kt, rat, t * 32, d), qop[d], x);
                y = mfma<T>(rows_op<DP>(vt, rat, t * 32, d), gop[d], y);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float w = __builtin_amdgcn_exp2f(x[e] * a.c - lse) *
                          (y[e] - delta);
                if (see == 1) {
                    const int j = k0 + t * 32 + e / 4 * 8 + lane / 32 * 4 +
                                  e % 4;
                    if (!view.sees(j)) w = 0.f;
                }
                x[e] = w;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const s16x8 op = pack8<T>(x, u * 8);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d)
                    acc[d] = mfma<T>(
                        cols_op<DP>(kt, cat, t * 32 + u * 16, d), op,
                        acc[d]);
            }
        }
    };
    // two buffers by name, so that reads of one are known not to touch
    // what is on its way into the other
    while (i < end) {
        step(kt0, vt0, kt1, vt1);
        if (++i >= end) break;
        step(kt1, vt1, kt0, vt0);
        ++i;
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            acc[d][e] = live ? acc[d][e] * a.scale : 0.f;
    if (SPLIT) {
        if (r < SG) store_sums<DP>(a.part_o + (row * a.splits + split) * DP,
                                   acc, lane);
        return;
    }
    // lanes without a row take part in the exchanges, and write nothing
    store_row<T, DP>((T *)a.dq + orow, acc, r < SG ? a.D : 0, lane);
}

// Adds the parts of dq in order: four columns of a row a thread.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_dq(const Args a)
{
    constexpr int PER = DP / 4;
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = e / PER;
    const int c = (int)(e - row * PER) * 4;
    if (row >= (long long)a.B * a.Hk * a.S * a.G || c >= a.D) return;
    const float *part = a.part_o + row * a.splits * DP + c;
    f32x4 x = {};
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i)
        x += *(const f32x4 *)(part + (long long)i * DP);
    const long long bh = row / (a.S * a.G);
    const int r = (int)(row - bh * (a.S * a.G)), qi = r / a.G;
    const int g = r - qi * a.G;
    const int b = (int)(bh / a.Hk), h = (int)(bh - (long long)b * a.Hk);
    typedef __attribute__((ext_vector_type(4))) T T4;
    T4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (T)x[j];
    *(T4 *)((T *)a.dq +
            (((long long)b * a.S + qi) * a.Hk * a.G + h * a.G + g) * a.D +
            c) = y;
}

// Rows that see any of keys k0..k1, as positions [p0, p1].
__device__ inline void rows_of(const Args &a, const Seq &s, int k0, int k1,
                               int &p0, int &p1)
{
    if (k1 > s.n - 1) k1 = s.n - 1;
    const bool first = k0 < a.sinks;
    p0 = a.causal ? k0 : first ? 0 : k0 - a.window + 1;
    p1 = first || a.window > s.n - k1 ? s.n - 1 : k1 + a.window - 1;
    if (k0 > k1) p1 = INT_MIN / 2;
    if (p0 < 0) p0 = 0;
    if (p0 < s.start) p0 = s.start;
    if (p1 > s.n - 1) p1 = s.n - 1;
    if (p1 > s.start + a.S - 1) p1 = s.start + a.S - 1;
}

// Rows [r0, r1) that see the block of keys from k0, and into how many parts of
// `piece` rows they are cut.
struct KeyRows {
    int r0, r1, piece, parts;
};
__device__ inline KeyRows key_rows(const Args &a, const Seq &s, int k0)
{
    KeyRows k = {0, 0, k0 < a.sinks && a.sink_blocks ? a.sink_rows
                                                     : a.splits_rows,
                 1};
    int p0, p1;
    rows_of(a, s, k0, k0 + a.keys - 1, p0, p1);
    if (p0 <= p1) {
        k.r0 = (p0 - s.start) * a.G;
        k.r1 = (p1 - s.start + 1) * a.G;
        k.parts = (int)(((long long)k.r1 - k.r0 + k.piece - 1) / k.piece);
    }
    return k;
}

// Parts of it that hold anything for the 32 keys from w0: where those are
// past the first tokens, no more than reach to the end of the last key's
// window.
__device__ inline int parts_of(const Args &a, const KeyRows &k, int k0,
                               int w0)
{
    if (k0 >= a.sinks || w0 < a.sinks) return k.parts;
    const long long rows = ((long long)k0 + a.keys + a.window) * a.G;
    const long long n = (rows + k.piece - 1) / k.piece;
    return n < k.parts ? (int)n : k.parts;
}

// Blocks of f32 sums of a head: the parts of first tokens' blocks, and of the
// others where those are cut.
__host__ __device__ inline int kv_slots(const Args &a)
{
    return a.sink_blocks * a.sink_splits +
           (a.splits > 1 ? (a.blocks - a.sink_blocks) * a.splits : 0);
}

// What dk and dv need of a tile's rows.
template <int KT>
struct RowData {
    __align__(16) float lse[KT];
    __align__(16) float delta[KT];
    __align__(16) int pos[KT];
};

// ---- backward: dk and dv ----
// A wave owns 32 keys; tiles of rows of q and dout stream by. Key blocks
// with first tokens are seen by all rows: they are split into parts of
// `splits_rows` rows whose f32 sums attn_join_kv adds in order, and so are
// the others where there are few blocks.
template <typename T, int DP, int NW>
__global__
__launch_bounds__(NW *WAVE, DP > 64 ? 2 : 3) void attn_dkv(const Args a)
{
    constexpr int KT = NW < 4 ? 32 : TILE;
    typedef Tile<DP, KT> Tile;
    typedef RowData<KT> RowData;
    __shared__ Tile qt0, qt1, gt0, gt1;
    __shared__ RowData rd0, rd1;
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int heads = a.B * a.Hk;
    int u = blockIdx.x / heads, blk, part;
    const int bh = blockIdx.x - u * heads, slot = u;
    if (u < a.sink_blocks * a.sink_splits) {
        blk = u / a.sink_splits;
        part = u - blk * a.sink_splits;
    } else {
        u -= a.sink_blocks * a.sink_splits;
        blk = u / a.splits;
        part = u - blk * a.splits;
        blk += a.sink_blocks;
    }
    const int b = bh / a.Hk, h = bh - b * a.Hk;
    const int SG = a.S * a.G;
    const Seq s = sequence(a, b);
    const int k0 = blk * NW * 32, w0 = k0 + wid * 32;
    const int key = w0 + lane % 32;
    const KeyRows kr = key_rows(a, s, k0);
    if (part >= kr.parts) return;  // the whole block
    const long long from = kr.r0 + (long long)part * kr.piece;
    const int r0 = (int)from;
    const int r1 = kr.r1 - from > kr.piece ? r0 + kr.piece : kr.r1;

    s16x8 kop[DP / 16], vop[DP / 16];
    {
        const long long at = key < a.T ? key : a.T - 1;
        const short *krow =
            (const short *)a.k + b * a.kb + at * a.ks + h * a.kh;
        const short *vrow =
            (const short *)a.v + b * a.vb + at * a.vs + h * a.vh;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            int d = i * 16 + lane / 32 * 8;
            d = d < a.D ? d : 0;
            kop[i] = *(const s16x8 *)(krow + d);
            vop[i] = *(const s16x8 *)(vrow + d);
        }
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const int d = i * 16 + lane / 32 * 8;
            if (key >= s.n || d >= a.D) kop[i] = vop[i] = s16x8{};
        }
    }
    // the rows that see this lane's key, as positions
    int plo = 0, phi = -1;
    if (key < s.n) rows_of(a, s, key, key, plo, phi);

    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = f32x16{};

    int rat = rows_at<DP>(lane), cat = cols_at<DP>(lane);
    // Where G divides the rows that the waves load at once, a lane's rows
    // are the same queries and heads of every tile, at the same offsets
    // from its first query.
    typedef Offsets<DP, NW, KT> Off;
    typedef Share<DP, NW, KT> Mine;
    const bool even = a.even && (!Off::WHOLE || Off::EACH % a.G == 0);
    Off qo, go;
    if (even) {
        qo.set(wid, lane, a.D, [&](int row) {
            const unsigned qi = row / a.G, g = row - qi * a.G;
            return qi * (unsigned)a.qs + g * (unsigned)a.qh;
        });
        go.set(wid, lane, a.D, [&](int row) {
            const unsigned qi = row / a.G, g = row - qi * a.G;
            return qi * (unsigned)a.gs + g * (unsigned)a.gh;
        });
    }
    const short *qbase =
        (const short *)a.q + b * a.qb + (long long)h * a.G * a.qh;
    const short *gbase =
        (const short *)a.dout + b * a.gb + (long long)h * a.G * a.gh;
    // a row past the last one repeats it: its lse takes its weight to 0
    auto send = [&](int t0, Tile &qt, Tile &gt, RowData &rd) {
        if (even && t0 + KT <= r1) {
            const int qi = t0 / a.G, step = Off::EACH / a.G;
            qo.send(qt, qbase + qi * a.qs, step * a.qs, wid);
            go.send(gt, gbase + qi * a.gs, step * a.gs, wid);
        } else {
            auto row = [&](int v) {
                const int r = t0 + Mine::row(v, wid, lane);
                return r < r1 ? r : r1 - 1;
            };
            send_tile<DP, NW, 1>(qt, wid, [&](int v) {
                const int r = row(v), qi = r / a.G, g = r - qi * a.G;
                return qbase + qi * a.qs + g * a.qh +
                       Mine::col(v, wid, lane, a.D);
            });
            send_tile<DP, NW, 1>(gt, wid, [&](int v) {
                const int r = row(v), qi = r / a.G, g = r - qi * a.G;
                return gbase + qi * a.gs + g * a.gh +
                       Mine::col(v, wid, lane, a.D);
            });
        }
        if (wid == 0) {
            const int r = t0 + lane;
            float l = __builtin_inff(), d = 0.f;
            int p = INT_MIN;
            if (r < r1) {
                l = a.lse[(long long)bh * SG + r];
                d = a.delta[(long long)bh * SG + r];
                p = s.start + r / a.G;
            }
            if (lane < KT) {
                rd.lse[lane] = l;
                rd.delta[lane] = d;
                rd.pos[lane] = p;
            }
        }
    };
    int t0 = r0;
    auto step = [&](const Tile &qt, const Tile &gt,
                    const RowData &rd, Tile &qn, Tile &gn,
                    RowData &rn) {
        landed();
        __syncthreads();
        if (t0 + KT < r1) send(t0 + KT, qn, gn, rn);
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
            const int f = t0 + t * 32;
            if (f >= r1) break;
            const int last = f + 31 < r1 ? f + 31 : r1 - 1;
            const int see = seen(a, s, s.start + f / a.G,
                                 s.start + last / a.G, w0, w0 + 31);
            if (see == 0) continue;
            // at 128 columns the sixteen places that follow from these two
            // are not kept in registers over the loop
            if (DP > 96) asm volatile("" : "+v"(rat), "+v"(cat));
            f32x16 x = {}, y = {};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                x = mfma<T>(rows_op<DP>(qt, rat, t * 32, d), kop[d], x);
                y = mfma<T>(rows_op<DP>(gt, rat, t * 32, d), vop[d], y);
            }
            // the products' operands are not read ahead across the steps:
            // there are no registers for them
            if (DP > 96) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int at = t * 32 + e4 * 8 + lane / 32 * 4;
                const f32x4 lse = *(const f32x4 *)&rd.lse[at];
                const f32x4 del = *(const f32x4 *)&rd.delta[at];
                float w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = __builtin_amdgcn_exp2f(x[e4 * 4 + j] * a.c -
                                                  lse[j]);
                if (see == 1) {
                    const i32x4 pos = *(const i32x4 *)&rd.pos[at];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool on = pos[j] >= plo && pos[j] <= phi;
                        w[j] = on ? w[j] : 0.f;
                        // w = 0 times what a hidden row holds is 0 too
                        y[e4 * 4 + j] = on ? y[e4 * 4 + j] : del[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[e4 * 4 + j] = w[j];
                    y[e4 * 4 + j] = w[j] * (y[e4 * 4 + j] - del[j]);
                }
            }
            if (DP > 96) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const s16x8 pop = pack8<T>(x, v * 8);
                const s16x8 sop = pack8<T>(y, v * 8);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) {
                    dv[d] = mfma<T>(
                        cols_op<DP>(gt, cat, t * 32 + v * 16, d), pop,
                        dv[d]);
                    dk[d] = mfma<T>(
                        cols_op<DP>(qt, cat, t * 32 + v * 16, d), sop,
                        dk[d]);
                }
            }
        }
    };
    if (t0 < r1) send(t0, qt0, gt0, rd0);
    while (t0 < r1) {
        step(qt0, gt0, rd0, qt1, gt1, rd1);
        if ((t0 += KT) >= r1) break;
        step(qt1, gt1, rd1, qt0, gt0, rd0);
        t0 += KT;
    }
    if (kr.parts > 1) {
        if (key >= a.T || part >= parts_of(a, kr, k0, w0)) return;
        const long long at =
            (((long long)bh * kv_slots(a) + slot) * NW * 32 + (key - k0)) *
            DP;
        store_sums<DP>(a.part_k + at, dk, lane);
        store_sums<DP>(a.part_v + at, dv, lane);
        return;
    }
    const long long at =
        (((long long)b * a.T + key) * a.Hk + h) * a.D;
    const int D = key < a.T ? a.D : 0;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][e] *= a.scale;
    store_row<T, DP>((T *)a.dk + at, dk, D, lane);
    store_row<T, DP>((T *)a.dv + at, dv, D, lane);
}

// Adds the parts of dk and dv: four columns of a key a thread, each wave of
// a block a quarter of the parts in order, then the quarters in order.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_kv(const Args a, int blocks)
{
    constexpr int PER = DP / 4;           // threads of a key
    __shared__ f32x4 sums[4][2][WAVE];
    const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
    const int each = a.keys * PER / WAVE;  // workgroups of a block of keys
    const int id = blockIdx.x / each, bh = id / blocks;
    const int blk = id - bh * blocks, k0 = blk * a.keys;
    const int e = (blockIdx.x - id * each) * WAVE + lane;
    const int key = k0 + e / PER, c = e % PER * 4;
    const int b = bh / a.Hk, h = bh - b * a.Hk;
    const KeyRows kr = key_rows(a, sequence(a, b), k0);
    if (kr.parts <= 1) return;  // written where it was summed
    const int parts = parts_of(a, kr, k0, key & ~31);
    const long long slot =
        blk < a.sink_blocks
            ? (long long)blk * a.sink_splits
            : (long long)a.sink_blocks * a.sink_splits +
                  (long long)(blk - a.sink_blocks) * a.splits;
    const long long part = (long long)a.keys * DP;
    const long long from = ((long long)bh * kv_slots(a) + slot) * part + e * 4;
    f32x4 x = {}, y = {};
    const int p1 = parts * (wid + 1) / 4;
#pragma unroll 8
    for (int i = parts * wid / 4; i < p1; ++i) {
        x += *(const f32x4 *)(a.part_k + from + i * part);
        y += *(const f32x4 *)(a.part_v + from + i * part);
    }
    sums[wid][0][lane] = x;
    sums[wid][1][lane] = y;
    __syncthreads();
    if (wid > 1 || key >= a.T || c >= a.D) return;
    // wave 0 writes dk, wave 1 dv
    x = sums[0][wid][lane];
#pragma unroll
    for (int i = 1; i < 4; ++i) x += sums[i][wid][lane];
    const float by = wid ? 1.f : a.scale;
    typedef __attribute__((ext_vector_type(4))) T T4;
    T4 z;
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = (T)(x[j] * by);
    const long long at = (((long long)b * a.T + key) * a.Hk + h) * a.D + c;
    *(T4 *)((T *)(wid ? a.dv : a.dk) + at) = z;
}

// ---- how the work is cut ----
constexpr int CUS = 256;
constexpr int FEW = 8;  // parts of a row that one thread still adds up
constexpr int FEW_KEYS = 32;

inline int dp_of(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

// Most key tiles that a block of `rows` rows visits.
long long most_tiles(const Args &a, int rows)
{
    long long keys = (rows + a.G - 1) / a.G;
    if (a.window < a.T)
        keys += (a.causal ? 1ll : 2ll) * a.window + a.sinks + 2 * KT;
    else
        keys = a.T;
    if (keys > a.T) keys = a.T;
    return (keys + KT - 1) / KT;
}

struct RowPlan {
    int waves, blocks, splits;
};

// Whether blocks are of 64 rows or keys and tiles of 32, instead of 128 and
// 64: what a block sees past each of its rows' windows is half as much,
// which pays where that is a good part of it. 6 sequences of 1999 tokens,
// 12 heads of 64, window 257, a training step: 136 us against 150; window
// 512, 4 x 4096 tokens of 16 heads: 320 both, 4096 tokens of 8/2 heads,
// forward: 22 against 18; window 1024, forward: 96 against 94.
bool narrow(const Args &a, long long n)
{
    return n > 128 && a.window < a.T &&
           (a.causal ? 1ll : 2ll) * a.window <= 384;
}

// Rows of a block: four waves of 32, or two, share each key tile; one where
// the rows fill no more. Where most places for blocks are left idle, the
// keys are split until there is a block for each, with at least eight tiles
// (2048 causal tokens, 16 heads of 64, 256 blocks for 768 places: dq 58 us
// whole, 36 + 7 us split and joined; with a window of 512 over 4096 tokens
// of 8/2 heads 26 us whole, 26 + 5 us split) or, of one wave, four.
RowPlan plan_rows(const Args &a, bool few)
{
    RowPlan p;
    const long long SG = (long long)a.S * a.G;
    p.waves = few && SG <= 32 ? 1 : narrow(a, SG) ? 2 : 4;
    p.blocks = (int)((SG + p.waves * 32 - 1) / (p.waves * 32));
    p.splits = 1;
    const long long all = (long long)p.blocks * a.B * a.Hk;
    const long long tiles = most_tiles(a, p.waves * 32);
    const int places =
        (p.waves == 1 ? 4 : (a.D > 64 ? 2 : 3) * (p.waves == 2 ? 2 : 1)) *
        CUS;
    if (all < (p.waves == 1 ? places : places / 2)) {
        long long n = (places + all - 1) / all;
        const long long least = p.waves == 1 ? 4 : 8;
        if (n > tiles / least) n = tiles / least;
        if (n > 1) p.splits = (int)n;
    }
    return p;
}

// dk and dv: where there are fewer blocks of keys than places for them, the
// rows that see a block are cut so that all places have one even share
// (s8192, 16/4 heads of 128, no mask: 256 blocks for 512 places, 1924 us
// uncut, 1131 us in halves). Where causal blocks of all lengths leave most
// places idle behind the longest, they are cut in thirds of a share (b2
// s4096, 16/4 heads of 128: 555 us in shares, 450 us in thirds), though the
// sums then take more of the memory's time (38 us there). Blocks are cut only
// where they are fewer than the places, so the parts are at most seven a
// place, whatever the lengths: 470 MB of f32 sums.
// The blocks with first tokens, which every row sees, are cut into eighths
// of the others' rows, so that they fill up what those leave at the end:
// 8192 tokens, 32/8 heads of 128, window 1024, has 504 blocks and 57 such
// eighths a head for 512 places.
void plan_dkv(Args &a)
{
    const long long SG = (long long)a.S * a.G;
    const bool window = a.window < a.T;
    // at 128 columns two waves' addresses would not fit the registers
    a.keys = narrow(a, a.T) && a.D <= 64 ? 64 : 128;
    a.blocks = (a.T + a.keys - 1) / a.keys;
    const long long sink =
        window
            ? ((a.sinks < a.T ? a.sinks : a.T) + a.keys - 1ll) / a.keys
            : 0;
    a.sink_blocks = (int)sink;
    long long rows =
        window ? (a.keys + (a.causal ? 1ll : 2ll) * a.window) * a.G : SG;
    if (rows > SG) rows = SG;
    const long long bh = (long long)a.B * a.Hk;
    const long long places =
        (a.D > 64 ? 2ll : 3ll) * (a.keys == 64 ? 2 : 1) * CUS;
    auto tiles = [](long long n) {  // at least 256 rows, whole tiles
        n = n < 256 ? 256 : n;
        return (n + KT - 1) / KT * KT;
    };
    // where causal and without a window, blocks see half of the rows
    const long long each = a.causal && !window ? rows / 2 : rows;
    const long long share = bh * a.blocks * each / places;
    const bool cut = each < rows ? rows > 2 * share : rows > share;
    const long long piece =
        tiles(!cut ? rows : each < rows ? share / 3 : share);
    a.splits_rows = (int)piece;
    a.splits = (int)((rows + piece - 1) / piece);
    a.sink_rows = a.splits_rows;
    a.sink_splits = 1;
    if (sink) {
        // no more than 1024 parts in all, or one each: their f32 sums take
        // 134 MB at most, however small the other blocks' pieces are (131072
        // tokens, 32/8 heads of 128, window 128, 1024 first tokens: 5.4 GB
        // if their pieces were cut as small)
        const long long most =
            bh * sink < 4 * CUS ? 4 * CUS / (bh * sink) : 1;
        long long n = tiles(rows / 8);
        if (n > piece) n = piece;
        if (n * most < SG) n = tiles((SG + most - 1) / most);
        a.sink_rows = (int)n;
        a.sink_splits = (int)((SG + n - 1) / n);
    }
}

long long kv_units(const Args &a)
{
    return (long long)a.sink_blocks * a.sink_splits +
           (long long)(a.blocks - a.sink_blocks) * a.splits;
}

bool kv_parts(const Args &a)
{
    return a.splits > 1 || (a.sink_blocks > 0 && a.sink_splits > 1);
}

template <typename T, int DP>
hipError_t launch_fwd(Args &a, const RowPlan &p, hipStream_t s)
{
    const long long n = (long long)a.B * a.Hk * p.blocks * p.splits;
    if (n * 64 * p.waves >= 1ll << 32) return hipErrorInvalidValue;
    const dim3 grid((unsigned)n);
    if (p.waves == 1) {
        if (p.splits > 1)
            attn_fwd<T, DP, 1, true><<<grid, 64, 0, s>>>(a);
        else
            attn_fwd<T, DP, 1, false><<<grid, 64, 0, s>>>(a);
    } else if (p.waves == 2) {
        if (p.splits > 1)
            attn_fwd<T, DP, 2, true><<<grid, 128, 0, s>>>(a);
        else
            attn_fwd<T, DP, 2, false><<<grid, 128, 0, s>>>(a);
    } else {
        if (p.splits > 1)
            attn_fwd<T, DP, 4, true><<<grid, 256, 0, s>>>(a);
        else
            attn_fwd<T, DP, 4, false><<<grid, 256, 0, s>>>(a);
    }
    if (p.splits > 1) {  // rows of few blocks, so few
        const long long rows = (long long)a.B * a.Hk * a.S * a.G;
        if (p.splits > FEW)
            attn_join<T><<<(unsigned)rows, 256, 0, s>>>(a, DP);
        else
            attn_join_few<T, DP>
                <<<(unsigned)((rows * (DP / 4) + 255) / 256), 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch_bwd(Args &a, hipStream_t s)
{
    const long long SG = (long long)a.S * a.G, bh = (long long)a.B * a.Hk;
    Args d = a;
    const RowPlan p = plan_rows(a, false);
    d.blocks = p.blocks;
    d.splits = p.splits;
    const long long near = a.causal ? a.window : 2ll * a.window - 1;
    d.few = a.T <= FEW_KEYS || near + a.sinks <= FEW_KEYS;
    const long long n = bh * d.blocks * d.splits, m = bh * kv_units(a);
    const bool parts = kv_parts(a);
    const int joined = a.splits > 1 ? a.blocks : a.sink_blocks;
    const long long j = parts ? bh * joined * (a.keys * (DP / 4) / WAVE) : 0;
    if (n * 256 >= 1ll << 32 || m * 256 >= 1ll << 32 || j * 256 >= 1ll << 32)
        return hipErrorInvalidValue;
    if (p.splits > 1) {
        if (p.waves == 2)
            attn_dq<T, DP, 2, true><<<(unsigned)n, 128, 0, s>>>(d);
        else
            attn_dq<T, DP, 4, true><<<(unsigned)n, 256, 0, s>>>(d);
        attn_join_dq<T, DP>
            <<<(unsigned)((bh * SG * (DP / 4) + 255) / 256), 256, 0, s>>>(d);
    } else if (p.waves == 2) {
        attn_dq<T, DP, 2, false><<<(unsigned)n, 128, 0, s>>>(d);
    } else {
        attn_dq<T, DP, 4, false><<<(unsigned)n, 256, 0, s>>>(d);
    }
    if (a.keys == 64)  // of at most 64 columns
        attn_dkv<T, DP <= 64 ? DP : 64, 2>
            <<<(unsigned)m, 128, 0, s>>>(a);
    else
        attn_dkv<T, DP, 4><<<(unsigned)m, 256, 0, s>>>(a);
    if (parts)
        attn_join_kv<T, DP><<<(unsigned)j, 256, 0, s>>>(a, joined);
    return hipGetLastError();
}

// dims: B, S, T, Hk, G, D, window, sinks, causal
void set_dims(Args &a, const long long *dims)
{
    a.B = (int)dims[0];
    a.S = (int)dims[1];
    a.T = (int)dims[2];
    a.Hk = (int)dims[3];
    a.G = (int)dims[4];
    a.D = (int)dims[5];
    a.window = (int)dims[6];
    a.sinks = (int)dims[7];
    a.causal = (int)dims[8];
}

// elements whose bytes a 32-bit offset reaches
bool near(long long n) { return n >= 0 && n < 1ll << 30; }

// the limits that the kernels' 32-bit positions, rows and offsets in a tile
// of keys rest on
bool fits(const long long *d)
{
    for (int i = 0; i < 6; ++i)
        if (d[i] < 1 || d[i] >= 1 << 30) return false;
    return d[1] * d[4] < 1 << 30 && d[0] * d[3] < 1 << 30 && d[5] <= 128 &&
           d[5] % 8 == 0 && d[6] >= 1 && d[6] <= 1 << 30 && d[7] >= 0 &&
           d[7] <= 1 << 30;
}

}  // namespace

extern "C" {

// Workspace bytes of the forward (0 where the keys are not split) or the
// backward; -1 where the sizes are out of range.
long long kf_attn_ws(const long long *dims, int backward)
{
    if (!fits(dims)) return -1;
    Args a = {};
    set_dims(a, dims);
    const long long rows = (long long)a.B * a.Hk * a.S * a.G;
    const int DP = dp_of(a.D);
    if (!backward) {
        const RowPlan p = plan_rows(a, true);
        return p.splits > 1 ? rows * p.splits * (DP + 2) * 4 : 0;
    }
    plan_dkv(a);
    long long n = (rows * 4 + 255) / 256 * 256;  // delta
    const RowPlan p = plan_rows(a, false);
    if (p.splits > 1) n += rows * p.splits * DP * 4;
    if (kv_parts(a))
        n += 2ll * a.B * a.Hk * kv_slots(a) * a.keys * DP * 4;
    return n;
}

// ptrs: q, k, v, out, lse and rest (or 0), lengths, starts, workspace
// strides: q (b s h), k, v in elements
hipError_t kf_attn_fwd(const uintptr_t *ptrs, const long long *dims,
                       const long long *st, float scale, int dtype,
                       void *stream)
{
    if (!fits(dims)) return hipErrorInvalidValue;
    Args a = {};
    set_dims(a, dims);
    a.q = (const void *)ptrs[0];
    a.k = (const void *)ptrs[1];
    a.v = (const void *)ptrs[2];
    a.out = (void *)ptrs[3];
    a.lse = (float *)ptrs[4];
    a.rest = (void *)ptrs[5];
    a.lengths = (const int *)ptrs[6];
    a.starts = (const int *)ptrs[7];
    a.qb = st[0], a.qs = st[1], a.qh = st[2];
    a.kb = st[3], a.ks = st[4], a.kh = st[5];
    a.vb = st[6], a.vs = st[7], a.vh = st[8];
    if (!near(a.ks * KT) || !near(a.vs * KT)) return hipErrorInvalidValue;
    a.scale = scale;
    a.c = scale * 1.44269504088896340736f;
    const RowPlan p = plan_rows(a, true);
    a.blocks = p.blocks;
    a.splits = p.splits;
    const int DP = dp_of(a.D);
    a.part_o = (float *)ptrs[8];
    a.part_ml =
        a.part_o + (long long)a.B * a.Hk * a.S * a.G * p.splits * DP;
    hipStream_t s = (hipStream_t)stream;
#define CASE(N)                                                             \
    if (DP == N)                                                            \
    return dtype == 1   ? launch_fwd<__bf16, N>(a, p, s)                    \
           : dtype == 2 ? launch_fwd<_Float16, N>(a, p, s)                  \
                        : hipErrorInvalidValue
    CASE(32);
    CASE(64);
    CASE(96);
    CASE(128);
#undef CASE
    return hipErrorInvalidValue;
}

// ptrs: q, k, v, out, lse, rest, lengths, starts, dout, dq, dk, dv,
//       workspace
// strides: q (b s h), k, v, dout in elements
hipError_t kf_attn_bwd(const uintptr_t *ptrs, const long long *dims,
                       const long long *st, float scale, int dtype,
                       void *stream)
{
    if (!fits(dims)) return hipErrorInvalidValue;
    Args a = {};
    set_dims(a, dims);
    a.q = (const void *)ptrs[0];
    a.k = (const void *)ptrs[1];
    a.v = (const void *)ptrs[2];
    a.o = (const void *)ptrs[3];
    a.lse = (float *)ptrs[4];
    a.orest = (const void *)ptrs[5];
    a.lengths = (const int *)ptrs[6];
    a.starts = (const int *)ptrs[7];
    a.dout = (const void *)ptrs[8];
    a.dq = (void *)ptrs[9];
    a.dk = (void *)ptrs[10];
    a.dv = (void *)ptrs[11];
    a.qb = st[0], a.qs = st[1], a.qh = st[2];
    a.kb = st[3], a.ks = st[4], a.kh = st[5];
    a.vb = st[6], a.vs = st[7], a.vh = st[8];
    if (!near(a.ks * KT) || !near(a.vs * KT)) return hipErrorInvalidValue;
    a.gb = st[9], a.gs = st[10], a.gh = st[11];
    a.scale = scale;
    a.c = scale * 1.44269504088896340736f;
    plan_dkv(a);
    a.even = 32 % a.G == 0 && near(a.qs * (KT / a.G) + a.qh * a.G) &&
             near(a.gs * (KT / a.G) + a.gh * a.G);
    const int DP = dp_of(a.D);
    const long long rows = (long long)a.B * a.Hk * a.S * a.G;
    a.delta = (float *)ptrs[12];
    const RowPlan p = plan_rows(a, false);
    a.part_o = a.delta + (rows * 4 + 255) / 256 * 64;
    a.part_k = a.part_o + (p.splits > 1 ? rows * p.splits * DP : 0);
    a.part_v = a.part_k + (long long)a.B * a.Hk * kv_slots(a) * a.keys * DP;
    hipStream_t s = (hipStream_t)stream;
#define CASE(N)                                                             \
    if (DP == N)                                                            \
    return dtype == 1   ? launch_bwd<__bf16, N>(a, s)                       \
           : dtype == 2 ? launch_bwd<_Float16, N>(a, s)                     \
                        : hipErrorInvalidValue
    CASE(32);
    CASE(64);
    CASE(96);
    CASE(128);
#undef CASE
    return hipErrorInvalidValue;
}

}  // extern "C"
