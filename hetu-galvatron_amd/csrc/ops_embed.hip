// Rows of an embedding table, and the table's gradient.
//
// Forward: out[n] = scale * weight[token(n) - first], zeros for tokens of other shards.  A copy with a lookup: bound by memory.
//
// Gradient: dW[r] = scale * sum over the places n of token r of grad[n].  Adding place by place with atomics would give sums that
// depend on timing, and a frequent token's row would be added to by thousands of places one after another.  Here places are
// ordered by token first, and sums are taken over pieces of that order:
//   index   one launch.  A workgroup owns the rows r with r % groups == its number (frequent tokens, which are neighbours in
//           vocabularies built by merges, spread over all of them), reads ALL tokens twice, counts its own and those of
//           workgroups before it -- so it knows where its part of the order begins without asking anyone -- and writes its places,
//           row by row and in the order of n within a row.
//   sum     a piece of `piece` neighbouring places of the order each: all pieces take equally long whatever the tokens are.
//           A row that lies in one piece is written; of a row that goes over the edge of a piece a partial sum is kept, at
//           most two of a piece.  The rest of the same launch fills the rows without places with zeros.
//   join    adds up the partial sums of a row, in order.
#include "ops_common.h"

#include <type_traits>

namespace {
using namespace ops;

constexpr int INDEX_WAVES = 16, INDEX_THREADS = 64 * INDEX_WAVES;
constexpr int INDEX_ROWS = 512;     // rows of a workgroup: a counter for each of them and each wave is 32 KB of LDS
constexpr int INDEX_AHEAD = 8;      // reads of tokens in flight for each lane
constexpr int INDEX_FOUND = 320;    // places of a wave that LDS keeps between counting and writing: 40 KB
constexpr uint32_t NONE = ~0u;      // a token without a row
constexpr int THREADS = 256;
// Rows that a unit of threads looks at for zeros: the lanes of a wave, or what a thread reads the counts of ahead.
constexpr int fill_rows(bool wide) { return wide ? 16 : 8; }

// Row numbers and where they go.
struct Index {
    int64_t n, first, rows;
    int32_t shift;       // log2 of the workgroups that share the rows
    int32_t per_group;   // rows of a workgroup
    int32_t *order;      // [n]  places by row
    int32_t *row;        // [n]  ... and the row of each
    int32_t *start;      // [groups * per_group]  of a row's places in `order`
    int32_t *count;      // [groups * per_group]
    int32_t *total;      // places with a row of this shard
    __device__ __forceinline__ int64_t slot(int64_t r) const { return (r & ((1 << shift) - 1)) * per_group + (r >> shift); }
};

// Bound by instructions: each workgroup looks at every token, some twelve of them a token and lane.  32768 tokens 12 us, 65536 20:
// of narrow tables with many tokens that is what counts, 65536 x 1024 bf16 into 32000 rows takes 74 us, 1.8 times its bytes' time.
template <typename I> __global__ __launch_bounds__(INDEX_THREADS) void embed_index_kernel(Index x, const I *__restrict__ tokens)
{
    __shared__ int32_t count[INDEX_WAVES][INDEX_ROWS];
    __shared__ uint2 found[INDEX_WAVES][INDEX_FOUND];   // place and row of a wave's first tokens that are the workgroup's
    __shared__ int32_t sums[INDEX_WAVES], before[INDEX_WAVES];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, group = blockIdx.x, mask = (1 << x.shift) - 1;
    for (int i = t; i < INDEX_WAVES * INDEX_ROWS; i += INDEX_THREADS) (&count[0][0])[i] = 0;
    __syncthreads();
    // A wave's tokens follow each other, so that its places are in order if it takes them in order.
    const int n = (int)x.n, each = (n + INDEX_THREADS - 1) / INDEX_THREADS * 64;
    const int from = min(wave * each, n), to = min(from + each, n);
    const uint32_t rows = (uint32_t)x.rows;
    const auto row_of = [&](int i) -> uint32_t {   // or NONE
        const int64_t r = (int64_t)tokens[i] - x.first;
        return (uint64_t)r < rows ? (uint32_t)r : NONE;
    };
    const uint64_t below = (1ull << lane) - 1;
    uint32_t lower = 0, n_found = 0;
    for (int at = from; at < to; at += 64 * INDEX_AHEAD) {
        uint32_t r[INDEX_AHEAD];
#pragma unroll
        for (int j = 0; j < INDEX_AHEAD; ++j) {
            const int i = at + 64 * j + lane;
            r[j] = row_of(min(i, n - 1));
            if (i >= to) r[j] = NONE;
        }
#pragma unroll
        for (int j = 0; j < INDEX_AHEAD; ++j) {
            const int of = r[j] == NONE ? INT32_MAX : (int)(r[j] & mask);
            lower += of < group;
            const uint64_t mine = __ballot(of == group);
            if (mine) {
                if (of == group) {
                    atomicAdd(&count[wave][r[j] >> x.shift], 1);
                    const uint32_t place = n_found + (uint32_t)__popcll(mine & below);
                    if (place < INDEX_FOUND) found[wave][place] = make_uint2((uint32_t)(at + 64 * j + lane), r[j]);
                }
                n_found += (uint32_t)__popcll(mine);
            }
        }
    }
    lower = wave_sum(lower);
    if (lane == 0) before[wave] = (int32_t)lower;
    __syncthreads();
    // counts -> where the places of each row and wave begin
    int32_t of_row = 0;
    if (t < x.per_group)
        for (int w = 0; w < INDEX_WAVES; ++w) {
            const int32_t c = count[w][t];
            count[w][t] = of_row;
            of_row += c;
        }
    int32_t upto = of_row;   // sum over the rows of a wave up to this one
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int32_t other = __shfl_up(upto, d);
        if (lane >= d) upto += other;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int32_t begin = upto - of_row;
    for (int w = 0; w < INDEX_WAVES; ++w) begin += before[w] + (w < wave ? sums[w] : 0);
    if (t < x.per_group) {
        for (int w = 0; w < INDEX_WAVES; ++w) count[w][t] += begin;
        x.start[(int64_t)group * x.per_group + t] = begin;
        x.count[(int64_t)group * x.per_group + t] = of_row;
    }
    if (group == mask && t == INDEX_THREADS - 1) *x.total = begin + of_row;   // (rows beyond per_group have no places)
    __syncthreads();
    const auto put = [&](uint32_t place, uint32_t row, bool mine) {
        const int local = mine ? (int)(row >> x.shift) : -1;
        uint64_t left = __ballot(mine);
        while (left) {   // one row at a time, of frequent tokens most often the only one
            const int leader = __builtin_ctzll(left);
            const int one = __builtin_amdgcn_readlane(local, leader);
            const uint64_t same = __ballot(local == one);
            int32_t to_place = 0;
            if (lane == leader) to_place = atomicAdd(&count[wave][one], (int)__popcll(same));
            to_place = __builtin_amdgcn_readlane(to_place, leader);
            if (local == one) {
                to_place += (int)__popcll(same & below);
                x.order[to_place] = (int32_t)place;
                x.row[to_place] = (int32_t)row;
            }
            left &= ~same;
        }
    };
    if (n_found <= INDEX_FOUND) {
        for (uint32_t i = 0; i < n_found; i += 64) {
            const bool mine = i + lane < n_found;
            const uint2 f = mine ? found[wave][i + lane] : make_uint2(0, 0);
            put(f.x, f.y, mine);
        }
        return;
    }
    for (int at = from; at < to; at += 64 * INDEX_AHEAD) {   // too many to be kept: look at all of them again
        uint32_t r[INDEX_AHEAD];
#pragma unroll
        for (int j = 0; j < INDEX_AHEAD; ++j) r[j] = row_of(min(at + 64 * j + lane, n - 1));
#pragma unroll
        for (int j = 0; j < INDEX_AHEAD; ++j) {
            const int i = at + 64 * j + lane;
            put((uint32_t)i, r[j], i < to && r[j] != NONE && (int)(r[j] & mask) == group);
        }
    }
}

struct Sum {
    Index index;
    int64_t dim;
    int32_t piece, pieces;
    int32_t unit;        // threads that share a row: a power of two
    int32_t accumulate, past;
    float scale;
    int64_t grad_stride, out_stride;
    float *partial;      // [pieces][2][dim]: of the row that began before the piece, of the one that goes on behind it
};

// A thread's columns: N from `col` on.  Where N does not divide the width, the last thread takes the last N, some of which are
// another's as well: both have the same sums for them.
struct Columns {
    int64_t col;
    int others;   // of them, at the front
    bool in;
};
template <int N> __device__ __forceinline__ Columns columns_of(int64_t dim, int unit)
{
    const int64_t col = ((int64_t)blockIdx.y * unit + threadIdx.x % unit) * N;
    return {col + N <= dim ? col : dim - N, col + N <= dim ? 0 : (int)(col + N - dim), col < dim};
}

template <typename O, int N> __device__ __forceinline__ void put_row(const Sum &s, typename O::raw *out, int64_t row, const Columns &at, const float (&acc)[N])
{
    typename O::raw *p = out + row * s.out_stride + at.col;
    float v[N];
    Pack<O, N> old;
    if (s.accumulate) old.load(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = s.accumulate ? fmaf(acc[i], s.scale, old[i]) : acc[i] * s.scale;
    old.set(v);
    old.store_from(p, s.accumulate ? at.others : 0);   // (what is added to is added to once)
}

// Bound by memory: 32768 places of 4096 bf16 added up and 128256 rows written in 217 us, 1.32 GB at 6.1 TB/s; 16384 places into 19008 rows of
// 5120 float32 in 66 us, 328 MB at 5.0 TB/s.  Sixteen rows are on their way to each thread, past the caches, since each is read once.
// WIDE: the threads that share a row are whole waves.  Then a wave's lanes read the numbers of 64 rows at once, which saves each row a
// wait for them.
template <typename T, typename O, int N, bool WIDE>
__global__ __launch_bounds__(THREADS) void embed_sum_kernel(Sum s, const typename T::raw *__restrict__ grad, typename O::raw *__restrict__ out)
{
    const Index &x = s.index;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / s.unit) + threadIdx.x / s.unit;
    const Columns at_columns = columns_of<N>(s.dim, s.unit);
    const int64_t col = at_columns.col;
    const bool in = at_columns.in;
    if (!WIDE && !in) return;
    if (unit >= s.pieces) {   // rows without places
        if (s.accumulate) return;
        const int64_t r0 = (unit - s.pieces) * fill_rows(WIDE);
        Pack<O, N> zeros;
        zeros.zero();
        if constexpr (WIDE) {
            uint64_t none = __ballot(lane < fill_rows(true) && r0 + lane < x.rows && x.count[x.slot(r0 + lane)] == 0);
            while (none) {
                typename O::raw *const p = out + (r0 + __builtin_ctzll(none)) * s.out_stride + col;
                if (in && s.past)
                    zeros.store_past(p);
                else if (in)
                    zeros.store(p);
                none &= none - 1;
            }
        } else {
#pragma unroll
            for (int i = 0; i < fill_rows(false); ++i)
                if (r0 + i < x.rows && x.count[x.slot(r0 + i)] == 0) zeros.store(out + (r0 + i) * s.out_stride + col);
        }
        return;
    }
    const int64_t total = *x.total, begin = unit * s.piece;
    if (begin >= total) return;
    const int64_t end = begin + s.piece < total ? begin + s.piece : total;
    const int32_t ahead = begin > 0 ? x.row[begin - 1] : -1, behind = end < total ? x.row[end] : -1;
    float acc[N];
    int32_t row = x.row[begin];
    bool from_ahead = row == ahead;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.0f;
    const auto put = [&](bool goes_on) {
        if (!in) return;
        if (from_ahead || goes_on) {
            float *p = s.partial + (unit * 2 + (from_ahead ? 0 : 1)) * s.dim + col;
            Pack<F32, N> v;
            v.set(acc);
            v.store(reinterpret_cast<F32::raw *>(p));
        } else
            put_row<O, N>(s, out, row, at_columns, acc);
    };
    constexpr int AHEAD = 16;
    int32_t rows_of = 0, places_of = 0;
    for (int64_t at = begin; at < end; at += AHEAD) {
        if (WIDE && ((at - begin) & 63) == 0) {
            const int64_t p = at + lane < end ? at + lane : end - 1;
            rows_of = x.row[p], places_of = x.order[p];
        }
        Pack<T, N> v[AHEAD];
        int32_t r[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            int32_t place;
            if constexpr (WIDE) {
                const int of = (int)((at - begin) & 63) + j;
                r[j] = __builtin_amdgcn_readlane(rows_of, of), place = __builtin_amdgcn_readlane(places_of, of);
            } else {
                const int64_t p = at + j < end ? at + j : end - 1;
                r[j] = x.row[p], place = x.order[p];
            }
            v[j].zero();
            if (in) v[j].load_past(grad + place * s.grad_stride + col);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (at + j >= end) break;
            if (r[j] != row) {
                put(false);
                row = r[j];
                from_ahead = false;
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += v[j][i];
        }
    }
    put(row == behind);
}

// A frequent token's row is a partial sum for each of its pieces, one after another: few columns a wave, so that many cores read
// them, and AHEAD reads at a time.  32768 tokens, the most frequent 5.9 % of them: 59 sums of 4096, 11 us; 14 with 2048 columns a
// workgroup and 8 reads.
constexpr int JOIN_UNIT = 64;
template <typename O, int N> __global__ __launch_bounds__(THREADS) void embed_join_kernel(Sum s, typename O::raw *__restrict__ out)
{
    const Index &x = s.index;
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / JOIN_UNIT) + threadIdx.x / JOIN_UNIT;
    const Columns at_columns = columns_of<N>(s.dim, JOIN_UNIT);
    const int64_t col = at_columns.col;
    const int64_t end = (unit + 1) * s.piece;
    if (!at_columns.in || end >= x.n) return;
    const int64_t total = *x.total;
    const int32_t row = x.row[end - 1], next = x.row[end];   // (read together; behind `total` they are any number)
    if (end >= total || row != next) return;
    const int64_t slot = x.slot(row), start = x.start[slot], stop = start + x.count[slot];
    if (start < unit * s.piece) return;   // began in a piece before: that one's
    float acc[N];
    Pack<F32, N> v;
    v.load(reinterpret_cast<const F32::raw *>(s.partial + (unit * 2 + 1) * s.dim + col));
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = v[i];
    const int64_t last = (stop - 1) / s.piece;
    constexpr int AHEAD = 16;
    for (int64_t u = unit + 1; u <= last; u += AHEAD) {
        Pack<F32, N> more[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) more[j].load(reinterpret_cast<const F32::raw *>(s.partial + (u + j < last ? u + j : last) * 2 * s.dim + col));
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (u + j <= last)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += more[j][i];
    }
    put_row<O, N>(s, out, row, at_columns, acc);
}

struct Rows {
    int64_t n, dim, rows, first;
    int32_t unit, each;   // threads that share a row, rows of such a unit
    int32_t token_type, past;
    float scale;
    int64_t weight_stride, out_stride;
};

// Bound by memory: 32768 tokens of 4096 bf16, half the table: 71 us, 350 MB at 4.9 TB/s, where calls follow each other; traced, each
// behind a wait, 77.  64 tokens of 1024: 3.0 us, a launch.
template <typename T, typename O, int N>
__global__ __launch_bounds__(THREADS) void embed_rows_kernel(Rows s, const void *__restrict__ tokens, const typename T::raw *__restrict__ weight,
                                                             typename O::raw *__restrict__ out)
{
    const int64_t unit = (int64_t)blockIdx.x * (THREADS / s.unit) + threadIdx.x / s.unit;
    const Columns at_columns = columns_of<N>(s.dim, s.unit);
    const int64_t col = at_columns.col;
    if (!at_columns.in) return;
    constexpr int AHEAD = 4;
    const int64_t begin = unit * s.each, end = begin + s.each < s.n ? begin + s.each : s.n;
    for (int64_t at = begin; at < end; at += AHEAD) {
        Pack<T, N> v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            v[j].zero();
            if (at + j < end) {
                const int64_t r = token_at(tokens, s.token_type, at + j) - s.first;
                if (r >= 0 && r < s.rows) v[j].load(weight + r * s.weight_stride + col);
            }
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (at + j < end) {
                float f[N];
#pragma unroll
                for (int i = 0; i < N; ++i) f[i] = v[j][i] * s.scale;
                Pack<O, N> o;
                o.set(f);
                if (s.past)
                    o.store_past(out + (at + j) * s.out_stride + col);
                else
                    o.store(out + (at + j) * s.out_stride + col);
            }
    }
}

// Whether an output of more than `most` bytes is written past the caches, the last of which has 256 MB.  Lookups from 128 MB on: of 268 MB
// 72 us, 80 through the caches.  Zeros of gradients from 512 MB on: of 1.05 GB the gradient takes 241 us, 282 through them, but of
// 263 MB 93 us, 78 through them.  Where rows do not begin with a line's 64 bytes the caches put lines together: 131 MB of zeros 29 us,
// 41 past them.
bool past_caches(const void *p, int64_t rows, int64_t dim, int64_t stride, int type, int64_t most)
{
    return rows * dim * size_of(type) > most && aligned(p, 64) && stride * size_of(type) % 64 == 0;
}

// Elements that a thread takes of a row at a time: 16 bytes of the smaller of the two types, one of rows that have less.
template <typename T, typename O> constexpr int AT_ONCE = T::VEC > O::VEC ? T::VEC : O::VEC;
int elements_at_once(int64_t dim, int type_a, int type_b)
{
    const int n = type_a == GDP_F32 && type_b == GDP_F32 ? AT_ONCE<F32, F32> : AT_ONCE<F16, F16>;
    return dim < n ? 1 : n;
}

// The threads that share a row: enough for all of it, a power of two so that units fill a workgroup.
int unit_of(int64_t dim, int n)
{
    int u = 1;
    while (u < THREADS && (int64_t)u * n < dim) u *= 2;
    return u;
}

template <typename F> int with_type(int t, F f)
{
    switch (t) {
    case GDP_F32: return f(F32{});
    case GDP_F16: return f(F16{});
    default: return f(BF16{});
    }
}
template <typename T, typename O, typename F> int with_count(int n, F f)
{
    return n == 1 ? f(std::integral_constant<int, 1>{}) : f(std::integral_constant<int, AT_ONCE<T, O>>{});
}

// Sizes of the order and of the partial sums, by which the workspace is laid out.
struct Layout {
    int shift, piece;
    int64_t per_group, pieces;
    size_t order, row, start, count, total, partial, bytes;
};

Layout layout_of(int64_t n, int64_t rows, int64_t dim)
{
    Layout l;
    l.shift = 0;
    while (l.shift < 8 && (1ll << l.shift) < rows) ++l.shift;
    while (ceil_div(rows, (int64_t)1 << l.shift) > INDEX_ROWS) ++l.shift;
    l.per_group = ceil_div(rows, (int64_t)1 << l.shift);
    // A longer piece keeps fewer partial sums, which the join adds up one after another; a shorter one fills the device.  Up to 1024
    // pieces do both: the gradient of 128256 x 4096 bf16 from 32768 tokens takes 240 us, 247 with 512, 251 with 2048 pieces.
    l.piece = 16;
    while (l.piece < 128 && n > 1024 * l.piece) l.piece *= 2;
    l.pieces = ceil_div(n, (int64_t)l.piece);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    l.order = take((size_t)n * 4);
    l.row = take((size_t)n * 4);
    l.start = take(((size_t)l.per_group << l.shift) * 4);
    l.count = take(((size_t)l.per_group << l.shift) * 4);
    l.total = take(4);
    l.partial = take((size_t)l.pieces * 2 * (size_t)dim * 4);
    l.bytes = at;
    return l;
}

// (grids of a few workgroups for each 4 tokens or 16 rows stay within 2^32 threads)
constexpr int64_t MOST_TOKENS = ((int64_t)1 << 26) - 4096, MOST_ROWS = (int64_t)1 << 27;
int check_sizes(int64_t n, int64_t rows, int64_t dim, int64_t first = 0)
{
    if (n < 0 || rows < 0 || dim < 0 || first < 0) return gdp_fail(GDP_E_BADARG, "gdp_embed: a size is negative");
    if (n > MOST_TOKENS || rows > MOST_ROWS || dim > (1 << 20))
        return gdp_fail(GDP_E_BADARG, "gdp_embed: more than 2^26 - 4096 tokens, 2^27 rows or 2^20 columns");
    return GDP_OK;
}

}  // namespace

extern "C" int gdp_embed_forward(const gdp_embed *e, void *stream)
{
    gdp_clear_error();
    if (!e) return gdp_fail(GDP_E_BADARG, "gdp_embed: null argument");
    if (const int rc = check_sizes(e->n, e->rows, e->dim, e->first)) return rc;
    if (!type_ok(e->weight_type) || !type_ok(e->out_type) || !token_type_ok(e->token_type))
        return gdp_fail(GDP_E_BADARG, "gdp_embed: unknown element type");
    if (e->n == 0 || e->dim == 0) return GDP_OK;
    if (!e->tokens || !e->out || (e->rows && !e->weight)) return gdp_fail(GDP_E_BADARG, "gdp_embed: null pointer");
    if (!rows_ok(e->rows, e->dim, e->weight_stride, false) || !rows_ok(e->n, e->dim, e->out_stride, true))
        return gdp_fail(GDP_E_BADARG, "gdp_embed: a row stride is negative, too large, or below the width of rows that are written");
    if (!aligned(e->weight, size_of(e->weight_type)) || !aligned(e->out, size_of(e->out_type)) ||
        !aligned(e->tokens, e->token_type == GDP_I64 ? 8 : 4))
        return gdp_fail(GDP_E_BADARG, "gdp_embed: a pointer is not aligned to its elements");
    const int n = elements_at_once(e->dim, e->weight_type, e->out_type);
    Rows s{e->n, e->dim, e->rows, e->first, unit_of(e->dim, n), 1, e->token_type, past_caches(e->out, e->n, e->dim, e->out_stride, e->out_type, 128 << 20), e->scale, e->weight_stride, e->out_stride};
    const int64_t across = ceil_div(e->dim, (int64_t)s.unit * n), per = THREADS / s.unit;
    if (ceil_div(e->n, per * 4) * across >= 2048) s.each = 4;   // rows in flight of a thread, where there are enough for all
    const int64_t blocks = ceil_div(e->n, per * s.each);
    return with_type(e->weight_type, [&](auto T) {
        return with_type(e->out_type, [&](auto O) {
            using TT = decltype(T);
            using OO = decltype(O);
            return with_count<TT, OO>(n, [&](auto N) {
                return launch("gdp_embed_forward", embed_rows_kernel<TT, OO, N.value>, dim3((unsigned)blocks, (unsigned)across), THREADS, 0, stream,
                              s, e->tokens, static_cast<const typename TT::raw *>(e->weight), static_cast<typename OO::raw *>(e->out));
            });
        });
    });
}

extern "C" int gdp_embed_grad_workspace(int64_t n, int64_t rows, int64_t dim, size_t *bytes)
{
    gdp_clear_error();
    if (!bytes) return gdp_fail(GDP_E_BADARG, "gdp_embed: null argument");
    if (const int rc = check_sizes(n, rows, dim)) return rc;
    *bytes = layout_of(n, rows, dim).bytes;
    return GDP_OK;
}

extern "C" int gdp_embed_backward(const gdp_embed_grad *e, void *stream)
{
    gdp_clear_error();
    if (!e) return gdp_fail(GDP_E_BADARG, "gdp_embed: null argument");
    if (const int rc = check_sizes(e->n, e->rows, e->dim, e->first)) return rc;
    if (!type_ok(e->grad_type) || !type_ok(e->out_type) || !token_type_ok(e->token_type))
        return gdp_fail(GDP_E_BADARG, "gdp_embed: unknown element type");
    if (e->rows == 0 || e->dim == 0 || (e->n == 0 && e->accumulate)) return GDP_OK;
    if ((e->n && (!e->tokens || !e->grad)) || !e->out || !e->workspace) return gdp_fail(GDP_E_BADARG, "gdp_embed: null pointer");
    if (!rows_ok(e->n, e->dim, e->grad_stride, false) || !rows_ok(e->rows, e->dim, e->out_stride, true))
        return gdp_fail(GDP_E_BADARG, "gdp_embed: a row stride is negative, too large, or below the width of rows that are written");
    if (!aligned(e->grad, size_of(e->grad_type)) || !aligned(e->out, size_of(e->out_type)) ||
        !aligned(e->tokens, e->token_type == GDP_I64 ? 8 : 4) || !aligned(e->workspace, 256))
        return gdp_fail(GDP_E_BADARG, "gdp_embed: a pointer is not aligned to its elements, or the workspace not to 256 bytes");
    const Layout l = layout_of(e->n, e->rows, e->dim);
    if (e->workspace_bytes < l.bytes) return gdp_fail(GDP_E_BADARG, "gdp_embed: the workspace is smaller than gdp_embed_grad_workspace says");
    char *const w = static_cast<char *>(e->workspace);
    const auto ints = [&](size_t at) { return reinterpret_cast<int32_t *>(w + at); };
    const Index x{e->n, e->first, e->rows, l.shift, (int32_t)l.per_group, ints(l.order), ints(l.row), ints(l.start), ints(l.count), ints(l.total)};
    int rc = e->token_type == GDP_I64
                 ? launch("gdp_embed_backward", embed_index_kernel<int64_t>, dim3(1u << l.shift), INDEX_THREADS, 0, stream, x, static_cast<const int64_t *>(e->tokens))
                 : launch("gdp_embed_backward", embed_index_kernel<int32_t>, dim3(1u << l.shift), INDEX_THREADS, 0, stream, x, static_cast<const int32_t *>(e->tokens));
    if (rc) return rc;
    const int n = elements_at_once(e->dim, e->grad_type, e->out_type);
    const Sum s{x, e->dim, l.piece, (int32_t)l.pieces, unit_of(e->dim, n), e->accumulate,
                past_caches(e->out, e->rows, e->dim, e->out_stride, e->out_type, 512 << 20), e->scale, e->grad_stride, e->out_stride,
                reinterpret_cast<float *>(w + l.partial)};
    const int64_t across = ceil_div(e->dim, (int64_t)s.unit * n), per = THREADS / s.unit;
    const int64_t units = l.pieces + (e->accumulate ? 0 : ceil_div(e->rows, (int64_t)fill_rows(s.unit >= 64)));
    return with_type(e->grad_type, [&](auto T) {
        return with_type(e->out_type, [&](auto O) {
            using TT = decltype(T);
            using OO = decltype(O);
            return with_count<TT, OO>(n, [&](auto N) {
                auto *const out = static_cast<typename OO::raw *>(e->out);
                auto kernel = embed_sum_kernel<TT, OO, N.value, false>;
                if constexpr (N.value > 1)   // (rows of single elements are shared by less than a wave)
                    if (s.unit >= 64) kernel = embed_sum_kernel<TT, OO, N.value, true>;
                const int rc = launch("gdp_embed_backward", kernel, dim3((unsigned)ceil_div(units, per), (unsigned)across), THREADS, 0, stream, s,
                                      static_cast<const typename TT::raw *>(e->grad), out);
                if (rc || l.pieces < 2) return rc;
                constexpr int J = N.value < 4 ? N.value : 4;
                return launch("gdp_embed_backward", embed_join_kernel<OO, J>, dim3((unsigned)ceil_div(l.pieces, (int64_t)(THREADS / JOIN_UNIT)), (unsigned)ceil_div(e->dim, (int64_t)JOIN_UNIT * J)),
                              THREADS, 0, stream, s, out);
            });
        });
    });
}
