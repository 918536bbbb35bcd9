// A block's output joined with the residual stream, with norms after the block and before the next one, and the gradients.
//
// All of it is bound by memory: a row is read once into registers, normed there (the mean of squares is taken around the mean, from
// the registers, so nothing cancels), joined, normed again and written.  Threads hold neighbouring elements of 16 bytes;
// a row has one to sixteen waves, and what a row's waves add up goes through LDS.
//
// Gradients.  With hat = (x - mean) * rstd and u = dy * weight,
//   dx = rstd * (u - mean(u * hat) * hat - mean(u))      (the last term with a mean only)
// first through the norm before, then the join, then gate and norm after.  Columns' sums (weights, biases, gate) stay in
// registers while a workgroup takes its rows one after another, and are written once a workgroup; a second kernel adds those up in
// a fixed order.
#include "ops_common.h"

#include <type_traits>

namespace {
using namespace ops;

struct Side {   // one norm
    int32_t form, type;
    float eps;
    const void *weight, *bias;
};

struct Join {
    int32_t n, dim, rows_per_gate;
    Side post, pre;
    int32_t gate_type;
    float residual_scale, block_scale, per_dim;
    int64_t residual_stride, block_stride, gate_stride, stream_stride, normed_stride;
    const void *gate;
    float4 *stats;
};

// Sums over the waves that share a row, at most W of them, in their order.  What a wave adds up lies in one of two places in turn, so
// that one barrier does: before a place is written again every wave has passed the barrier behind its reads.
template <int W> struct RowSums {
    __align__(16) float of_wave[2][2][W < 4 ? 4 : W];
};
template <int W, int N> __device__ __forceinline__ void row_sums(float (&v)[N], RowSums<W> &shared, int &turn)
{
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) shared.of_wave[turn][i][threadIdx.x >> 6] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[i] += shared.of_wave[turn][i][w];   // 0 of waves that are not there
        }
        turn ^= 1;
    }
}
template <int W> __device__ __forceinline__ void row_sums_begin(RowSums<W> &shared)
{
    if constexpr (W > 1) {
        if (threadIdx.x < 4 * W) (&shared.of_wave[0][0][0])[threadIdx.x] = 0.0f;
        __syncthreads();
    }
}

template <int E> __device__ __forceinline__ void row_of_weights(const void *p, int type, int64_t at, float (&w)[E], float idle)
{
    if (!p) {
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = idle;
    } else if (type == GDP_F32) {
        Pack<F32, E> v;
        v.load(static_cast<const F32::raw *>(p) + at);
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = v[i];
    } else {
        Pack<BF16, E> v;   // (f16 has the same size)
        v.load(static_cast<const BF16::raw *>(p) + at);
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = type == GDP_BF16 ? v[i] : F16::up(v.raw(i));
    }
}

// A thread's columns: E from `col` on, K times.  Where E does not divide the width (TAIL), the last thread takes the last E, the first
// `others` of which are another's: it leaves them out of sums and does not write them.  A thread behind the row's end has E others.
template <int K, int E, bool TAIL> struct Columns {
    int col[K], others[K];
    bool in[K];
    __device__ __forceinline__ Columns(int t, int threads, int dim)
    {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            col[k] = (k * threads + t) * E;
            in[k] = col[k] < dim;
            others[k] = in[k] ? 0 : E;
            if (TAIL && in[k] && col[k] + E > dim) {
                others[k] = col[k] + E - dim;
                col[k] = dim - E;
            }
        }
    }
    __device__ __forceinline__ bool own(int k, int i) const { return TAIL ? i >= others[k] : in[k]; }
    __device__ __forceinline__ int from(int k) const { return TAIL ? others[k] : 0; }   // the first that is written
};

// Mean and 1 / deviation of a row of which a thread holds x[K][E].
template <int W, int K, int E, bool TAIL>
__device__ __forceinline__ float2 statistics(const float (&x)[K][E], const Columns<K, E, TAIL> &c, int form, float eps, float per_dim, RowSums<W> &shared, int &turn)
{
    float mean = 0.0f;
    float sum[1] = {0.0f};
    if (form == GDP_NORM_LAYER) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < E; ++i) sum[0] += c.own(k, i) ? x[k][i] : 0.0f;
        row_sums<W, 1>(sum, shared, turn);
        mean = sum[0] * per_dim;
    }
    sum[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float d = c.own(k, i) ? x[k][i] - mean : 0.0f;
            sum[0] = fmaf(d, d, sum[0]);
        }
    row_sums<W, 1>(sum, shared, turn);
    return make_float2(mean, 1.0f / sqrtf(fmaf(sum[0], per_dim, eps)));
}

// At most W waves to a row, K times E elements to a thread; R rows to a workgroup where W is 1.  16384 x 4096 bf16 with both norms and a
// gate: 108 us, 537 MB at 5.0 TB/s; 65536 x 1024 102 us; 8 x 4096 4.4 us, a launch and two barriers.  Rows below 512 elements of 16 bits leave
// lanes of their wave idle: 65536 x 128 36 us, 2.6 times its bytes' time.
template <typename T, typename S, int W, int K, int E, bool TAIL, int R>
__global__ __launch_bounds__(64 * W * R) void norm_forward_kernel(Join a, const typename S::raw *__restrict__ residual, const typename T::raw *__restrict__ block,
                                                                  typename S::raw *__restrict__ stream, typename T::raw *__restrict__ normed)
{
    __shared__ RowSums<W> shared;
    int turn = 0;
    const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x, threads = W == 1 ? 64 : blockDim.x;
    const int row = blockIdx.x * R + (W == 1 ? threadIdx.x >> 6 : 0);
    if (W == 1 && row >= a.n) return;
    row_sums_begin(shared);
    const Columns<K, E, TAIL> c(t, threads, a.dim);
    const auto &col = c.col;
    const auto &in = c.in;
    Pack<S, E> r[K];
    Pack<T, E> b[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        r[k].zero();
        b[k].zero();
        if (in[k]) {
            if (block) b[k].load(block + (int64_t)row * a.block_stride + col[k]);
            r[k].load(residual + (int64_t)row * a.residual_stride + col[k]);
        }
    }
    float x[K][E];
    float4 stats = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) x[k][i] = b[k][i];
    if (block) {
        if (a.post.form != GDP_NORM_NONE) {
            const float2 s = statistics<W, K, E, TAIL>(x, c, a.post.form, a.post.eps, a.per_dim, shared, turn);
            stats.x = s.x, stats.y = s.y;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (in[k]) {
                    float w[E], add[E];
                    row_of_weights<E>(a.post.weight, a.post.type, col[k], w, 1.0f);
                    row_of_weights<E>(a.post.bias, a.post.type, col[k], add, 0.0f);
#pragma unroll
                    for (int i = 0; i < E; ++i) x[k][i] = fmaf((x[k][i] - s.x) * s.y, w[i], add[i]);
                }
        }
        if (a.gate) {
            const int64_t g = (row / a.rows_per_gate) * a.gate_stride;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (in[k]) {
                    float w[E];
                    row_of_weights<E>(a.gate, a.gate_type, g + col[k], w, 1.0f);
#pragma unroll
                    for (int i = 0; i < E; ++i) x[k][i] *= w[i];
                }
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < E; ++i) x[k][i] = block ? fmaf(r[k][i], a.residual_scale, x[k][i] * a.block_scale) : r[k][i] * a.residual_scale;
        if (stream && in[k]) {
            r[k].set(x[k]);
            r[k].store_from(stream + (int64_t)row * a.stream_stride + col[k], c.from(k));
        }
    }
    if (a.pre.form != GDP_NORM_NONE) {
        const float2 s = statistics<W, K, E, TAIL>(x, c, a.pre.form, a.pre.eps, a.per_dim, shared, turn);
        stats.z = s.x, stats.w = s.y;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (in[k]) {
                float w[E], add[E];
                row_of_weights<E>(a.pre.weight, a.pre.type, col[k], w, 1.0f);
                row_of_weights<E>(a.pre.bias, a.pre.type, col[k], add, 0.0f);
#pragma unroll
                for (int i = 0; i < E; ++i) x[k][i] = fmaf((x[k][i] - s.x) * s.y, w[i], add[i]);
                b[k].set(x[k]);
                b[k].store_from(normed + (int64_t)row * a.normed_stride + col[k], c.from(k));
            }
    }
    if (a.stats && t == 0) a.stats[row] = stats;
}

enum { PRE_W, PRE_B, POST_W, POST_B, GATE, COLUMNS };   // sums over rows

struct Back {
    int32_t n, dim, rows_per_gate;
    int32_t groups, per_group;   // workgroups; rows of one, or (split_gates) workgroups that share the rows of a gate
    int32_t split_gates, gate_type;
    Side post, pre;
    float residual_scale, block_scale, per_dim;
    int64_t stream_stride, block_stride, grad_normed_stride, grad_stream_stride, gate_stride, grad_residual_stride, grad_block_stride;
    const void *gate;
    const float4 *stats;
    float *partial;              // [sums that are asked for][groups][dim]
    float *of[COLUMNS];          // where each of those begins, or null
    void *grad_gate;             // written where a workgroup has all rows of its gates, and there are several
};

// The rows of a workgroup.  Each gate's rows go to `per_group` workgroups, or a workgroup has the rows of whole gates.
__device__ __forceinline__ void rows_of(const Back &a, int group, int &from, int &to)
{
    if (a.split_gates) {
        const int gate = group / a.per_group, q = group % a.per_group, each = (a.rows_per_gate + a.per_group - 1) / a.per_group;
        from = gate * a.rows_per_gate + min(q * each, a.rows_per_gate);
        to = gate * a.rows_per_gate + min((q + 1) * each, a.rows_per_gate);
    } else {
        from = min(group * a.per_group, a.n);
        to = min(from + a.per_group, a.n);
    }
}

// A row of weights, for each row of the gradient.  HOLD: a thread keeps what it needs of them packed, in the block's 16 bits, so that four
// rows of weights, five sums of columns and a row that is read ahead fit 168 registers, with which 12 waves are on a core.
// Otherwise (float32, mixed types, more than 12 waves with biases) they are read again for each row, H at a time, from the caches: kept unpacked they
// would take the registers of the sums.
template <typename T, int K, int E, bool TAIL, bool HOLD> struct Weights {
    static constexpr int H = E < 4 ? E : 4;
    const void *p;
    int type;
    float idle;
    Pack<T, E> w[HOLD ? K : 1];
    __device__ __forceinline__ void read(const void *row, int type_, const Columns<K, E, TAIL> &c, float idle_)
    {
        p = row, type = type_, idle = idle_;
        if constexpr (HOLD) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float f[E];
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = idle;
                w[k].set(f);
                if (p && c.in[k]) w[k].load(static_cast<const typename T::raw *>(p) + c.col[k]);
            }
        }
    }
    // Tells the compiler that they may have changed: it would unpack, or read, them once for all rows.
    __device__ __forceinline__ void hold(int &again)
    {
        if constexpr (HOLD) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < Pack<T, E>::WORDS; ++i) asm volatile("" : "+v"(w[k].w[i]));
        } else {
            again = 0;
            asm volatile("" : "+s"(again));
        }
    }
    __device__ __forceinline__ void get(int k, int h, int again, const Columns<K, E, TAIL> &c, float (&f)[H]) const
    {
        if constexpr (HOLD) {
#pragma unroll
            for (int i = 0; i < H; ++i) f[i] = w[k][h + i];
        } else
            row_of_weights<H>(c.in[k] ? p : nullptr, type, c.col[k] + h + again, f, idle);
    }
};

// 16384 x 4096 bf16 (mean of squares, gate) in 168 us, 805 MB at 4.8 TB/s; 16384 x 3584 with mean, biases, a gate for each of 4 sequences and a
// float32 stream in 215 us and 6 for the sums, 1.06 GB at 4.9 TB/s.
// Above 8192 elements (K = 2) sums and a row do not fit the registers and some are spilled: 8192 x 12288 bf16 601 us, 2.4 times its
// bytes' time, x 16384 1070 us, 3.2 times.
// BIAS: with sums for biases.
template <typename T, typename S, bool HOLD, bool BIAS, int W, int K, int E, bool TAIL>
__global__ __launch_bounds__(64 * W, W <= 4 ? 4 : W <= 12 ? 3 : 1) void norm_backward_kernel(Back a, const typename S::raw *__restrict__ stream, const typename T::raw *__restrict__ block,
                                                               const typename T::raw *__restrict__ grad_normed, const typename S::raw *__restrict__ grad_stream,
                                                               typename S::raw *__restrict__ grad_residual, typename T::raw *__restrict__ grad_block)
{
    __shared__ RowSums<W> shared;
    int turn = 0;
    const int t = threadIdx.x, threads = blockDim.x;
    row_sums_begin(shared);
    const Columns<K, E, TAIL> c(t, threads, a.dim);
    const auto &col = c.col;
    const auto &in = c.in;
    float sums[COLUMNS][K][E];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int q = 0; q < COLUMNS; ++q)
#pragma unroll
            for (int i = 0; i < E; ++i) sums[q][k][i] = 0.0f;
    int from, to;
    rows_of(a, blockIdx.x, from, to);
    using Row = Weights<T, K, E, TAIL, HOLD>;
    constexpr int H = Row::H;
    Row pre_w, post_w, post_b, gate;
    const bool post = a.post.form != GDP_NORM_NONE;
    pre_w.read(a.pre.weight, a.pre.type, c, 1.0f);
    post_w.read(post ? a.post.weight : nullptr, a.post.type, c, 1.0f);
    post_b.read(post ? a.post.bias : nullptr, a.post.type, c, 0.0f);
    gate.read(nullptr, 0, c, 1.0f);
    struct Read {
        Pack<S, E> r[K], ds[K];
        Pack<T, E> b[K], dh[K];
        float4 stats;
    };
    const auto read = [&](Read &o, int row) {
        o.stats = a.stats[row];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            o.r[k].zero(), o.ds[k].zero(), o.b[k].zero(), o.dh[k].zero();
            if (in[k]) {
                if (grad_normed) {
                    o.dh[k].load(grad_normed + (int64_t)row * a.grad_normed_stride + col[k]);
                    o.r[k].load(stream + (int64_t)row * a.stream_stride + col[k]);
                }
                if (grad_stream) o.ds[k].load(grad_stream + (int64_t)row * a.grad_stream_stride + col[k]);
                if (block) o.b[k].load(block + (int64_t)row * a.block_stride + col[k]);
            }
        }
    };
    // Of 5 to 12 waves one workgroup is on a core, with registers to read a row ahead (16384 rows of 4096 bf16: 170 us, 181 with
    // two workgroups that wait in turn and 128 registers); of fewer there are several (65536 of 1024: 179, 188 ahead).
    constexpr bool AHEAD = K == 1 && (W == 8 || W == 12);
    Read next;
    if (AHEAD && from < to) read(next, from);
    for (int row = from; row < to; ++row) {
        const int64_t g = row / a.rows_per_gate;
        if (a.gate && (row == from || row % a.rows_per_gate == 0))
            gate.read(static_cast<const char *>(a.gate) + g * a.gate_stride * (a.gate_type == GDP_F32 ? 4 : 2), a.gate_type, c, 1.0f);
        int again = 0;
        pre_w.hold(again), post_w.hold(again), post_b.hold(again), gate.hold(again);
        if (!AHEAD) read(next, row);
        Read now = next;
        if (AHEAD && row + 1 < to) read(next, row + 1);
        auto &r = now.r, &ds = now.ds;
        auto &b = now.b, &dh = now.dh;
        const float4 stats = now.stats;
        float d[K][E];   // of the stream
        if (grad_normed) {
            float mean[2] = {0.0f, 0.0f};   // of u * hat, of u
            const auto hat = [&](int k, int i) { return (r[k][i] - stats.z) * stats.w; };
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int h = 0; h < E; h += H) {
                    float w[H];
                    pre_w.get(k, h, again, c, w);
#pragma unroll
                    for (int i = h; i < h + H; ++i) {
                        const float y = c.own(k, i) ? dh[k][i] : 0.0f;
                        sums[PRE_W][k][i] = fmaf(y, hat(k, i), sums[PRE_W][k][i]);
                        if (BIAS) sums[PRE_B][k][i] += y;
                        d[k][i] = y * w[i - h];
                        mean[0] = fmaf(d[k][i], hat(k, i), mean[0]);
                        mean[1] += d[k][i];
                    }
                }
            row_sums<W, 2>(mean, shared, turn);
            mean[0] *= a.per_dim;
            mean[1] *= a.pre.form == GDP_NORM_LAYER ? a.per_dim : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < E; ++i) d[k][i] = c.own(k, i) ? fmaf(d[k][i] - hat(k, i) * mean[0] - mean[1], stats.w, ds[k][i]) : 0.0f;
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < E; ++i) d[k][i] = c.own(k, i) ? ds[k][i] : 0.0f;
        }
        if (grad_residual) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (in[k]) {
                    float f[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) f[i] = d[k][i] * a.residual_scale;
                    r[k].set(f);
                    r[k].store_from(grad_residual + (int64_t)row * a.grad_residual_stride + col[k], c.from(k));
                }
        }
        if (block) {
            float mean[2] = {0.0f, 0.0f};
            const auto hat = [&](int k, int i) { return post ? (b[k][i] - stats.x) * stats.y : b[k][i]; };
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int h = 0; h < E; h += H) {
                    float w[H], add[H], of_gate[H];
                    post_w.get(k, h, again, c, w), post_b.get(k, h, again, c, add), gate.get(k, h, again, c, of_gate);
#pragma unroll
                    for (int i = h; i < h + H; ++i) {
                        float dn = d[k][i] * a.block_scale;
                        sums[GATE][k][i] = fmaf(dn, fmaf(hat(k, i), w[i - h], add[i - h]), sums[GATE][k][i]);
                        dn *= of_gate[i - h];
                        sums[POST_W][k][i] = fmaf(dn, hat(k, i), sums[POST_W][k][i]);
                        if (BIAS) sums[POST_B][k][i] += dn;
                        d[k][i] = dn * w[i - h];
                        mean[0] = fmaf(d[k][i], hat(k, i), mean[0]);
                        mean[1] += d[k][i];
                    }
                }
            if (post) {
                row_sums<W, 2>(mean, shared, turn);
                mean[0] *= a.per_dim;
                mean[1] *= a.post.form == GDP_NORM_LAYER ? a.per_dim : 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) d[k][i] = (d[k][i] - hat(k, i) * mean[0] - mean[1]) * stats.y;
            }
            if (grad_block) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (in[k]) {
                        b[k].set(d[k]);
                        b[k].store_from(grad_block + (int64_t)row * a.grad_block_stride + col[k], c.from(k));
                    }
            }
            if (a.grad_gate && (row + 1) % a.rows_per_gate == 0) {   // the last row of a gate, all of whose rows are this workgroup's
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        if (c.own(k, i)) down_any(a.grad_gate, a.gate_type, g * a.dim + col[k] + i, sums[GATE][k][i]);
                        sums[GATE][k][i] = 0.0f;
                    }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < COLUMNS; ++q)
        if (a.of[q]) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (in[k]) {
                    Pack<F32, E> v;
                    v.set(sums[q][k]);
                    v.store_from(reinterpret_cast<F32::raw *>(a.of[q] + (int64_t)blockIdx.x * a.dim + col[k]), c.from(k));
                }
        }
}

// out[g][col] = sum of `rows` rows of partial sums, in their order: 32 sums of a 32nd each, joined in order.
struct Add {
    const float *from;
    void *to;
    int32_t rows, groups, type;
};
struct Adds {
    Add of[COLUMNS];
    int64_t dim;
};
constexpr int ADD_COLUMNS = 32, ADD_ROWS = 32;
__global__ __launch_bounds__(ADD_COLUMNS *ADD_ROWS) void norm_add_kernel(Adds a)
{
    __shared__ float part[ADD_ROWS][ADD_COLUMNS];
    const Add &o = a.of[blockIdx.z];
    const int c = threadIdx.x % ADD_COLUMNS, q = threadIdx.x / ADD_COLUMNS;
    const int64_t col = (int64_t)blockIdx.x * ADD_COLUMNS + c, group = blockIdx.y;
    if (group >= o.groups) return;
    float sum = 0.0f;
    if (col < a.dim) {
        const float *p = o.from + group * o.rows * a.dim + col;
        const int each = (o.rows + ADD_ROWS - 1) / ADD_ROWS, from = q * each, to = min(from + each, o.rows);
#pragma unroll 8
        for (int r = from; r < to; ++r) sum += p[r * a.dim];
    }
    part[q][c] = sum;
    __syncthreads();
    if (q == 0 && col < a.dim) {
        for (int i = 1; i < ADD_ROWS; ++i) sum += part[i][c];
        down_any(o.to, o.type, group * a.dim + col, sum);
    }
}

// ---- host ----
constexpr int64_t MOST_ROWS = (int64_t)1 << 22;   // of 1024 threads a workgroup, a grid of less than 2^32

int check_side(const gdp_norm_params &p, const char *what)
{
    if (p.form != GDP_NORM_NONE && p.form != GDP_NORM_RMS && p.form != GDP_NORM_LAYER) return gdp_fail(GDP_E_BADARG, what);
    if (p.form == GDP_NORM_NONE) return GDP_OK;
    if (!type_ok(p.type) || !(p.eps >= 0.0f) || !aligned(p.weight, size_of(p.type)) || !aligned(p.bias, size_of(p.type))) return gdp_fail(GDP_E_BADARG, what);
    return GDP_OK;
}
int check_sizes(int64_t n, int64_t dim, int type, int stream_type)
{
    if (n < 0 || dim < 1 || n >= MOST_ROWS || dim > GDP_MAX_NORM_DIM) return gdp_fail(GDP_E_BADARG, "gdp_norm: needs less than 2^22 rows of 1 to GDP_MAX_NORM_DIM columns");
    if (!type_ok(type) || !type_ok(stream_type) || (stream_type != type && stream_type != GDP_F32))
        return gdp_fail(GDP_E_BADARG, "gdp_norm: unknown element type, or a stream that is neither of the block's type nor float32");
    return GDP_OK;
}
int check_rows(const void *p, int64_t n, int64_t dim, int64_t stride, int type, bool written)
{
    if (!p) return GDP_OK;
    if (!rows_ok(n, dim, stride, written)) return gdp_fail(GDP_E_BADARG, "gdp_norm: a row stride is negative, too large, or below the width of rows that are written");
    if (!aligned(p, size_of(type))) return gdp_fail(GDP_E_BADARG, "gdp_norm: a pointer is not aligned to its elements");
    return GDP_OK;
}
int check_gate(const void *gate, int64_t gates, int64_t stride, int type, int64_t n, int64_t dim)
{
    if (!gate) return GDP_OK;
    if (gates < 1 || (n && n % gates)) return gdp_fail(GDP_E_BADARG, "gdp_norm: the number of gates must divide the number of rows");
    if (!type_ok(type)) return gdp_fail(GDP_E_BADARG, "gdp_norm: unknown element type");
    return check_rows(gate, gates, dim, stride, type, false);
}

template <typename F> int with_types(int type, int stream_type, F f)
{
    if (type == GDP_F32) return f(F32{}, F32{});
    if (type == GDP_BF16) return stream_type == GDP_F32 ? f(BF16{}, F32{}) : f(BF16{}, BF16{});
    return stream_type == GDP_F32 ? f(F16{}, F32{}) : f(F16{}, F16{});
}
template <int N> using Int = std::integral_constant<int, N>;

// f(most waves of a row, times that a thread's elements repeat, elements, whether they do not divide the width, threads): 16 bytes of the
// block's type a thread, 16 waves at most; rows of less than 16 bytes an element a thread.
template <int E, bool TAIL, bool FEW = true, typename F> int with_waves(int64_t dim, F f)   // FEW: there may be 8 waves or less
{
    using Tail = std::integral_constant<bool, TAIL>;
    const int waves = (int)ceil_div(dim, (int64_t)64 * E);
    if constexpr (FEW)
        if (waves <= 1) return f(Int<1>{}, Int<1>{}, Int<E>{}, Tail{}, 64);
    if constexpr (E > 1) {
        if constexpr (FEW) {
            if (waves <= 4) return f(Int<4>{}, Int<1>{}, Int<E>{}, Tail{}, 64 * waves);
            if (waves <= 8) return f(Int<8>{}, Int<1>{}, Int<E>{}, Tail{}, 64 * waves);
        }
        if (waves <= 12) return f(Int<12>{}, Int<1>{}, Int<E>{}, Tail{}, 64 * waves);
        if (waves <= 16) return f(Int<16>{}, Int<1>{}, Int<E>{}, Tail{}, 64 * waves);
        if constexpr (E == 8) {
            if (waves <= 24) return f(Int<12>{}, Int<2>{}, Int<E>{}, Tail{}, 64 * (int)ceil_div(waves, 2));
            return f(Int<16>{}, Int<2>{}, Int<E>{}, Tail{}, 64 * (int)ceil_div(waves, 2));
        }
    }
    return gdp_fail(GDP_E_BADARG, "gdp_norm: too wide");   // (not reached: 4 and 1 elements a thread are for narrower rows)
}
template <int E, typename F> int with_columns(int64_t dim, F f)
{
    if (dim < E) return with_waves<1, false>(dim, f);
    // (of float32 twice that where 16 waves do not reach otherwise: fewer repetitions, whose sums are kept in registers)
    if constexpr (E == 4)
        if (dim > 64 * 16 * 4) return dim % 8 ? with_waves<8, true, false>(dim, f) : with_waves<8, false, false>(dim, f);
    return dim % E ? with_waves<E, true>(dim, f) : with_waves<E, false>(dim, f);
}

static_assert(GDP_MAX_NORM_DIM <= 64 * 16 * 8 * 2, "the widest row fits");
Side side_of(const gdp_norm_params &p) { return {p.form, p.type, p.eps, p.weight, p.bias}; }

// How many workgroups take the rows of a gradient, and how: the rows of each of several gates are shared by some workgroups,
// or, where gates are many, a workgroup has the rows of whole gates.
struct Shares {
    int64_t groups, per_group;
    bool split_gates;
};
Shares shares_of(int64_t n, int64_t dim, int64_t gates)
{
    if (n == 0) return {0, 0, false};
    // Of 16-bit types as many workgroups as are resident together, by their registers 16 waves on a core of up to 4 waves each, else 12: each
    // writes its sums of columns, and one more than that would run alone at the end.  Waves are counted as of 512 columns; float32 up to 4096
    // columns has 256 a wave, so there are up to four times the workgroups that are resident: 16384 x 1024 91 us, 8192 x 2048 91, 8192 x 4096 170,
    // 1.1, 1.1 and 1.0 times their bytes' time.  Where rows are few each workgroup has one, and the sums weigh as much as the rows: 2048
    // x 1024 bf16 21 us, 4 times its bytes' time.
    const int64_t waves = ceil_div(dim, (int64_t)512), most = 256 * (waves <= 4 ? 16 / waves : waves <= 12 ? 12 / waves : 1);
    const int64_t rows = gates > 1 ? n / gates : 1, units = n / rows;
    if (gates > 1 && gates <= most / 2 && rows > 1) {
        const int64_t q = most / gates < rows ? most / gates : rows;
        return {gates * q, q, true};
    }
    const int64_t each = ceil_div(units, most);
    return {ceil_div(units, each), each * rows, false};
}

}  // namespace

extern "C" int gdp_norm_forward(const gdp_norm *p, void *queue)
{
    gdp_clear_error();
    if (!p) return gdp_fail(GDP_E_BADARG, "gdp_norm: null argument");
    if (const int rc = check_sizes(p->n, p->dim, p->type, p->stream_type)) return rc;
    if (const int rc = check_side(p->post, "gdp_norm: post: unknown form or type, eps below 0, or a pointer that is not aligned")) return rc;
    if (const int rc = check_side(p->pre, "gdp_norm: pre: unknown form or type, eps below 0, or a pointer that is not aligned")) return rc;
    if (const int rc = check_gate(p->gate, p->gates, p->gate_stride, p->gate_type, p->n, p->dim)) return rc;
    if (p->n == 0) return GDP_OK;   // (pointers to no rows may be null)
    if (!p->block && (p->post.form != GDP_NORM_NONE || p->gate)) return gdp_fail(GDP_E_BADARG, "gdp_norm: a norm or a gate of a block that is not given");
    if (!p->residual || (p->pre.form == GDP_NORM_NONE) != !p->normed || (!p->normed && !p->stream)) return gdp_fail(GDP_E_BADARG, "gdp_norm: null pointer, or an output that nothing is written to");
    if (const int rc = check_rows(p->residual, p->n, p->dim, p->residual_stride, p->stream_type, false)) return rc;
    if (const int rc = check_rows(p->block, p->n, p->dim, p->block_stride, p->type, false)) return rc;
    if (const int rc = check_rows(p->stream, p->n, p->dim, p->stream_stride, p->stream_type, true)) return rc;
    if (const int rc = check_rows(p->normed, p->n, p->dim, p->normed_stride, p->type, true)) return rc;
    if (!aligned(p->stats, 16)) return gdp_fail(GDP_E_BADARG, "gdp_norm: stats must be aligned to 16 bytes");
    const Join j{(int32_t)p->n, (int32_t)p->dim, (int32_t)(p->gate ? p->n / p->gates : p->n), side_of(p->post), side_of(p->pre), p->gate_type, p->residual_scale, p->block_scale, 1.0f / (float)p->dim,
                 p->residual_stride, p->block_stride, p->gate_stride, p->stream_stride, p->normed_stride, p->gate, reinterpret_cast<float4 *>(p->stats)};
    return with_types(p->type, p->stream_type, [&](auto T, auto S) {
        using TT = decltype(T);
        using SS = decltype(S);
        return with_columns<TT::VEC>(p->dim, [&](auto W, auto K, auto E, auto TAIL, int threads) {
            constexpr int R = W.value == 1 ? 4 : 1;
            return launch("gdp_norm_forward", norm_forward_kernel<TT, SS, W.value, K.value, E.value, TAIL.value, R>, dim3((unsigned)ceil_div(p->n, (int64_t)R)), threads * R, 0, queue,
                          j, static_cast<const typename SS::raw *>(p->residual), static_cast<const typename TT::raw *>(p->block), static_cast<typename SS::raw *>(p->stream),
                          static_cast<typename TT::raw *>(p->normed));
        });
    });
}

extern "C" int gdp_norm_grad_workspace(int64_t n, int64_t dim, int64_t gates, size_t *bytes)
{
    gdp_clear_error();
    if (!bytes) return gdp_fail(GDP_E_BADARG, "gdp_norm: null argument");
    if (const int rc = check_sizes(n, dim, GDP_F32, GDP_F32)) return rc;
    if (gates < 0 || (gates && n % gates)) return gdp_fail(GDP_E_BADARG, "gdp_norm: the number of gates must divide the number of rows");
    *bytes = round_up((size_t)COLUMNS * shares_of(n, dim, gates).groups * dim * 4, 256);
    return GDP_OK;
}

extern "C" int gdp_norm_backward(const gdp_norm_grad *p, void *queue)
{
    gdp_clear_error();
    if (!p) return gdp_fail(GDP_E_BADARG, "gdp_norm: null argument");
    if (const int rc = check_sizes(p->n, p->dim, p->type, p->stream_type)) return rc;
    if (const int rc = check_side(p->post, "gdp_norm: post: unknown form or type, eps below 0, or a pointer that is not aligned")) return rc;
    if (const int rc = check_side(p->pre, "gdp_norm: pre: unknown form or type, eps below 0, or a pointer that is not aligned")) return rc;
    if (p->n && !p->block && (p->post.form != GDP_NORM_NONE || p->gate || p->grad_block)) return gdp_fail(GDP_E_BADARG, "gdp_norm: a norm, a gate or a gradient of a block that is not given");
    if (const int rc = check_gate(p->gate, p->gates, p->gate_stride, p->gate_type, p->n, p->dim)) return rc;
    if ((p->grad_gate && !p->gate) || ((p->grad_pre_weight || p->grad_pre_bias) && p->pre.form == GDP_NORM_NONE) ||
        ((p->grad_post_weight || p->grad_post_bias) && p->post.form == GDP_NORM_NONE))
        return gdp_fail(GDP_E_BADARG, "gdp_norm: a gradient of something that is not given");
    if (p->n && (!p->stats || (p->pre.form == GDP_NORM_NONE) != !p->grad_normed || (p->grad_normed && !p->stream) || !p->workspace)) return gdp_fail(GDP_E_BADARG, "gdp_norm: null pointer");
    const struct { const void *p; int64_t stride; int type; bool written; } all[] = {
        {p->stream, p->stream_stride, p->stream_type, false}, {p->block, p->block_stride, p->type, false}, {p->grad_normed, p->grad_normed_stride, p->type, false},
        {p->grad_stream, p->grad_stream_stride, p->stream_type, false}, {p->grad_residual, p->grad_residual_stride, p->stream_type, true}, {p->grad_block, p->grad_block_stride, p->type, true}};
    for (const auto &a : all) {
        if (const int rc = check_rows(a.p, p->n, p->dim, a.stride, a.type, a.written)) return rc;
        }
    if (!aligned(p->stats, 16)) return gdp_fail(GDP_E_BADARG, "gdp_norm: stats must be aligned to 16 bytes");
    const int64_t gates = p->gate ? p->gates : 0;
    const Shares shares = shares_of(p->n, p->dim, gates);
    if (!aligned(p->workspace, 256) || p->workspace_bytes < round_up((size_t)COLUMNS * shares.groups * p->dim * 4, 256))
        return gdp_fail(GDP_E_BADARG, "gdp_norm: the workspace is smaller than gdp_norm_grad_workspace says, or not aligned to 256 bytes");
    Back b{(int32_t)p->n, (int32_t)p->dim, (int32_t)(gates ? p->n / gates : p->n), (int32_t)shares.groups, (int32_t)shares.per_group, shares.split_gates, p->gate_type,
           side_of(p->post), side_of(p->pre), p->residual_scale, p->block_scale, 1.0f / (float)p->dim, p->stream_stride, p->block_stride, p->grad_normed_stride,
           p->grad_stream_stride, p->gate_stride, p->grad_residual_stride, p->grad_block_stride, p->gate, reinterpret_cast<const float4 *>(p->stats),
           static_cast<float *>(p->workspace), {}, nullptr};
    Adds adds{};
    adds.dim = p->dim;
    void *const outs[COLUMNS] = {p->grad_pre_weight, p->grad_pre_bias, p->grad_post_weight, p->grad_post_bias, p->grad_gate};
    const int types[COLUMNS] = {p->pre.type, p->pre.type, p->post.type, p->post.type, p->gate_type};
    unsigned count = 0, most = 1;
    for (int c = 0; c < COLUMNS; ++c) {
        if (!outs[c]) continue;
        const bool several = c == GATE && gates > 1;   // a sum for each gate, not one over all rows
        if (several && !shares.split_gates && p->n) {
            b.grad_gate = outs[c];
            continue;
        }
        b.of[c] = b.partial + (int64_t)count * shares.groups * p->dim;
        adds.of[count++] = {b.of[c], outs[c], (int32_t)(several ? shares.per_group : shares.groups), (int32_t)(several ? gates : 1), types[c]};
        if (several) most = (unsigned)gates;
    }
    const auto of_type = [&](const void *w, int type) { return !w || type == p->type; };
    const bool packed = of_type(p->pre.weight, p->pre.type) && of_type(p->post.weight, p->post.type) && of_type(p->post.bias, p->post.type) && of_type(p->gate, p->gate_type);
    const int rc = p->n == 0 ? GDP_OK : with_types(p->type, p->stream_type, [&](auto T, auto S) {
        using TT = decltype(T);
        using SS = decltype(S);
        return with_columns<TT::VEC>(p->dim, [&](auto W, auto K, auto E, auto TAIL, int threads) {
            const auto run = [&](auto HOLD, auto BIAS) {
                return launch("gdp_norm_backward", norm_backward_kernel<TT, SS, HOLD.value, BIAS.value, W.value, K.value, E.value, TAIL.value>, dim3((unsigned)shares.groups), threads, 0,
                              queue, b, static_cast<const typename SS::raw *>(p->stream), static_cast<const typename TT::raw *>(p->block),
                              static_cast<const typename TT::raw *>(p->grad_normed), static_cast<const typename SS::raw *>(p->grad_stream),
                              static_cast<typename SS::raw *>(p->grad_residual), static_cast<typename TT::raw *>(p->grad_block));
            };
            const bool bias = p->grad_pre_bias || p->grad_post_bias;
            if constexpr (sizeof(typename TT::raw) == 2 && K.value == 1 && E.value > 1) {
                if (packed && !bias) return run(std::true_type{}, std::false_type{});
                if constexpr (W.value <= 12)
                    if (packed) return run(std::true_type{}, std::true_type{});
            }
            return bias ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});
        });
    });
    if (rc) return rc;
    const unsigned across = (unsigned)ceil_div(p->dim, (int64_t)ADD_COLUMNS);
    return count ? launch("gdp_norm_backward", norm_add_kernel, dim3(across, most, count), ADD_COLUMNS * ADD_ROWS, 0, queue, adds) : GDP_OK;
}
