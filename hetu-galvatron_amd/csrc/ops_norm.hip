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

// Mean and 1 / deviation of a row of which a thread holds x[K][E].
template <int W, int K, int E>
__device__ __forceinline__ float2 statistics(const float (&x)[K][E], const bool (&in)[K], int form, float eps, float per_dim, RowSums<W> &shared, int &turn)
{
    float mean = 0.0f;
    float sum[1] = {0.0f};
    if (form == GDP_NORM_LAYER) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < E; ++i) sum[0] += x[k][i];   // 0 outside
        row_sums<W, 1>(sum, shared, turn);
        mean = sum[0] * per_dim;
    }
    sum[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float d = in[k] ? x[k][i] - mean : 0.0f;
            sum[0] = fmaf(d, d, sum[0]);
        }
    row_sums<W, 1>(sum, shared, turn);
    return make_float2(mean, 1.0f / sqrtf(fmaf(sum[0], per_dim, eps)));
}

// At most W waves to a row, K times E elements to a thread; R rows to a workgroup where W is 1.
template <typename T, typename S, int W, int K, int E, int R>
__global__ __launch_bounds__(64 * W * R) void norm_forward_kernel(Join a, const typename S::raw *__restrict__ residual, const typename T::raw *__restrict__ block,
                                                                  typename S::raw *__restrict__ stream, typename T::raw *__restrict__ normed)
{
    __shared__ RowSums<W> shared;
    int turn = 0;
    const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x, threads = W == 1 ? 64 : blockDim.x;
    const int row = blockIdx.x * R + (W == 1 ? threadIdx.x >> 6 : 0);
    if (W == 1 && row >= a.n) return;
    row_sums_begin(shared);
    bool in[K];
    int col[K];
    Pack<S, E> r[K];
    Pack<T, E> b[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        col[k] = (k * threads + t) * E;
        in[k] = col[k] < a.dim;
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
            const float2 s = statistics<W, K, E>(x, in, a.post.form, a.post.eps, a.per_dim, shared, turn);
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
            r[k].store(stream + (int64_t)row * a.stream_stride + col[k]);
        }
    }
    if (a.pre.form != GDP_NORM_NONE) {
        const float2 s = statistics<W, K, E>(x, in, a.pre.form, a.pre.eps, a.per_dim, shared, turn);
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
                b[k].store(normed + (int64_t)row * a.normed_stride + col[k]);
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

template <typename T, typename S, int W, int K, int E>
__global__ __launch_bounds__(64 * W, W <= 8 ? 4 : 1) void norm_backward_kernel(Back a, const typename S::raw *__restrict__ stream, const typename T::raw *__restrict__ block,
                                                               const typename T::raw *__restrict__ grad_normed, const typename S::raw *__restrict__ grad_stream,
                                                               typename S::raw *__restrict__ grad_residual, typename T::raw *__restrict__ grad_block)
{
    __shared__ RowSums<W> shared;
    int turn = 0;
    const int t = threadIdx.x, threads = blockDim.x;
    row_sums_begin(shared);
    bool in[K];
    int col[K];
    float sums[COLUMNS][K][E];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        col[k] = (k * threads + t) * E;
        in[k] = col[k] < a.dim;
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
            for (int i = 0; i < E; ++i) sums[c][k][i] = 0.0f;
    }
    int from, to;
    rows_of(a, blockIdx.x, from, to);
    for (int row = from; row < to; ++row) {
        Pack<S, E> r[K], ds[K];
        Pack<T, E> b[K], dh[K];
        const float4 stats = a.stats[row];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            r[k].zero(), ds[k].zero(), b[k].zero(), dh[k].zero();
            if (in[k]) {
                if (grad_normed) {
                    dh[k].load(grad_normed + (int64_t)row * a.grad_normed_stride + col[k]);
                    r[k].load(stream + (int64_t)row * a.stream_stride + col[k]);
                }
                if (grad_stream) ds[k].load(grad_stream + (int64_t)row * a.grad_stream_stride + col[k]);
                if (block) b[k].load(block + (int64_t)row * a.block_stride + col[k]);
            }
        }
        float d[K][E];   // of the stream
        if (grad_normed) {
            float hat[K][E], mean[2] = {0.0f, 0.0f};   // of u * hat, of u
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float w[E];
#pragma unroll
                for (int i = 0; i < E; ++i) w[i] = 0.0f;
                if (in[k]) row_of_weights<E>(a.pre.weight, a.pre.type, col[k], w, 1.0f);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    hat[k][i] = (r[k][i] - stats.z) * stats.w;
                    sums[PRE_W][k][i] = fmaf(dh[k][i], hat[k][i], sums[PRE_W][k][i]);
                    sums[PRE_B][k][i] += dh[k][i];
                    d[k][i] = dh[k][i] * w[i];
                    mean[0] = fmaf(d[k][i], hat[k][i], mean[0]);
                    mean[1] += d[k][i];
                }
            }
            row_sums<W, 2>(mean, shared, turn);
            mean[0] *= a.per_dim;
            mean[1] *= a.pre.form == GDP_NORM_LAYER ? a.per_dim : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < E; ++i) d[k][i] = in[k] ? fmaf(d[k][i] - hat[k][i] * mean[0] - mean[1], stats.w, ds[k][i]) : 0.0f;
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < E; ++i) d[k][i] = ds[k][i];
        }
        if (grad_residual) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (in[k]) {
                    float f[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) f[i] = d[k][i] * a.residual_scale;
                    r[k].set(f);
                    r[k].store(grad_residual + (int64_t)row * a.grad_residual_stride + col[k]);
                }
        }
        if (block) {
            float hat[K][E], mean[2] = {0.0f, 0.0f};   // of u * hat, of u
            const int64_t g = row / a.rows_per_gate;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float w[E], add[E], gate[E];
#pragma unroll
                for (int i = 0; i < E; ++i) w[i] = 1.0f, add[i] = 0.0f, gate[i] = 1.0f;
                if (in[k]) {
                    if (a.post.form != GDP_NORM_NONE) {
                        row_of_weights<E>(a.post.weight, a.post.type, col[k], w, 1.0f);
                        row_of_weights<E>(a.post.bias, a.post.type, col[k], add, 0.0f);
                    }
                    row_of_weights<E>(a.gate, a.gate_type, g * a.gate_stride + col[k], gate, 1.0f);
                }
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    float dn = d[k][i] * a.block_scale;
                    hat[k][i] = a.post.form != GDP_NORM_NONE ? (b[k][i] - stats.x) * stats.y : b[k][i];
                    const float n = a.post.form != GDP_NORM_NONE ? fmaf(hat[k][i], w[i], add[i]) : b[k][i];
                    sums[GATE][k][i] = fmaf(dn, n, sums[GATE][k][i]);
                    dn *= gate[i];
                    sums[POST_W][k][i] = fmaf(dn, hat[k][i], sums[POST_W][k][i]);
                    sums[POST_B][k][i] += dn;
                    d[k][i] = dn * w[i];
                    mean[0] = fmaf(d[k][i], hat[k][i], mean[0]);
                    mean[1] += d[k][i];
                }
            }
            if (a.post.form != GDP_NORM_NONE) {
                row_sums<W, 2>(mean, shared, turn);
                mean[0] *= a.per_dim;
                mean[1] *= a.post.form == GDP_NORM_LAYER ? a.per_dim : 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) d[k][i] = (d[k][i] - hat[k][i] * mean[0] - mean[1]) * stats.y;
            }
            if (grad_block) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (in[k]) {
                        b[k].set(d[k]);
                        b[k].store(grad_block + (int64_t)row * a.grad_block_stride + col[k]);
                    }
            }
            if (a.grad_gate && (row + 1) % a.rows_per_gate == 0) {   // the last row of a gate, all of whose rows are this workgroup's
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        if (in[k]) down_any(a.grad_gate, a.gate_type, g * a.dim + col[k] + i, sums[GATE][k][i]);
                        sums[GATE][k][i] = 0.0f;
                    }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c)
        if (a.of[c]) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (in[k]) {
                    Pack<F32, E> v;
                    v.set(sums[c][k]);
                    v.store(reinterpret_cast<F32::raw *>(a.of[c] + (int64_t)blockIdx.x * a.dim + col[k]));
                }
        }
}

// out[g][col] = sum of `rows` rows of partial sums, in their order: 16 sums of a sixteenth each, joined in order.
struct Add {
    const float *from;
    void *to;
    int32_t rows, groups, type;
};
struct Adds {
    Add of[COLUMNS];
    int64_t dim;
};
constexpr int ADD_COLUMNS = 64, ADD_ROWS = 16;
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

// Whether all rows can be taken in 16 bytes: of `E` elements each.
struct Wide {
    int64_t dim;
    int e;
    bool ok;
    void rows(const void *p, int64_t stride, int type)
    {
        const int need = e * size_of(type) < 16 ? e * size_of(type) : 16;
        if (p && row_alignment(p, stride, type) < need) ok = false;
    }
};
Wide wide_for(int64_t dim, int type) { return {dim, 16 / size_of(type), dim % (16 / size_of(type)) == 0}; }

template <typename F> int with_types(int type, int stream_type, F f)
{
    if (type == GDP_F32) return f(F32{}, F32{});
    if (type == GDP_BF16) return stream_type == GDP_F32 ? f(BF16{}, F32{}) : f(BF16{}, BF16{});
    return stream_type == GDP_F32 ? f(F16{}, F32{}) : f(F16{}, F16{});
}
template <int N> using Int = std::integral_constant<int, N>;

// f(most waves of a row, times that a thread's elements repeat, threads): 16 bytes a thread, 16 waves at most.
template <int E, typename F> int with_waves(int64_t dim, F f)
{
    const int waves = (int)ceil_div(dim, (int64_t)64 * E);
    if (waves <= 1) return f(Int<1>{}, Int<1>{}, 64);
    if (waves <= 4) return f(Int<4>{}, Int<1>{}, 64 * waves);
    if (waves <= 8) return f(Int<8>{}, Int<1>{}, 64 * waves);
    if (waves <= 16) return f(Int<16>{}, Int<1>{}, 64 * waves);
    if constexpr (E == 8) return f(Int<16>{}, Int<2>{}, 64 * (int)ceil_div(waves, 2));
    if constexpr (E == 4) return f(Int<16>{}, Int<4>{}, 64 * (int)ceil_div(waves, 4));
    if constexpr (E == 1) return f(Int<16>{}, Int<16>{}, 64 * (int)ceil_div(waves, 16));
}
static_assert(GDP_MAX_NORM_DIM <= 64 * 16 * 16, "the widest row fits");

Side side_of(const gdp_norm_params &p) { return {p.form, p.type, p.eps, p.weight, p.bias}; }

// How many workgroups take the rows of a gradient, and how: the rows of each of several gates are shared by some workgroups,
// or, where gates are many, a workgroup has the rows of whole gates.
struct Shares {
    int64_t groups, per_group;
    bool split_gates;
};
constexpr int64_t MOST_GROUPS = 512;
Shares shares_of(int64_t n, int64_t gates)
{
    if (n == 0) return {0, 0, false};
    const int64_t rows = gates > 1 ? n / gates : 1, units = n / rows;
    if (gates > 1 && gates <= MOST_GROUPS / 2 && rows > 1) {
        const int64_t q = MOST_GROUPS / gates < rows ? MOST_GROUPS / gates : rows;
        return {gates * q, q, true};
    }
    const int64_t each = ceil_div(units, MOST_GROUPS);
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
    Wide wide = wide_for(p->dim, p->type);
    wide.rows(p->residual, p->residual_stride, p->stream_type);
    wide.rows(p->block, p->block_stride, p->type);
    wide.rows(p->stream, p->stream_stride, p->stream_type);
    wide.rows(p->normed, p->normed_stride, p->type);
    wide.rows(p->gate, p->gate_stride, p->gate_type);
    for (const gdp_norm_params *s : {&p->post, &p->pre})
        if (s->form != GDP_NORM_NONE) wide.rows(s->weight, 0, s->type), wide.rows(s->bias, 0, s->type);
    const Join j{(int32_t)p->n, (int32_t)p->dim, (int32_t)(p->gate ? p->n / p->gates : p->n), side_of(p->post), side_of(p->pre), p->gate_type, p->residual_scale, p->block_scale, 1.0f / (float)p->dim,
                 p->residual_stride, p->block_stride, p->gate_stride, p->stream_stride, p->normed_stride, p->gate, reinterpret_cast<float4 *>(p->stats)};
    return with_types(p->type, p->stream_type, [&](auto T, auto S) {
        using TT = decltype(T);
        using SS = decltype(S);
        const auto run = [&](auto E) {
            return with_waves<E.value>(p->dim, [&](auto W, auto K, int threads) {
                constexpr int R = W.value == 1 ? 4 : 1;
                return launch("gdp_norm_forward", norm_forward_kernel<TT, SS, W.value, K.value, E.value, R>, dim3((unsigned)ceil_div(p->n, (int64_t)R)), threads * R, 0, queue, j,
                              static_cast<const typename SS::raw *>(p->residual), static_cast<const typename TT::raw *>(p->block), static_cast<typename SS::raw *>(p->stream),
                              static_cast<typename TT::raw *>(p->normed));
            });
        };
        return wide.ok ? run(Int<TT::VEC>{}) : run(Int<1>{});
    });
}

extern "C" int gdp_norm_grad_workspace(int64_t n, int64_t dim, int64_t gates, size_t *bytes)
{
    gdp_clear_error();
    if (!bytes) return gdp_fail(GDP_E_BADARG, "gdp_norm: null argument");
    if (const int rc = check_sizes(n, dim, GDP_F32, GDP_F32)) return rc;
    if (gates < 0 || (gates && n % gates)) return gdp_fail(GDP_E_BADARG, "gdp_norm: the number of gates must divide the number of rows");
    *bytes = round_up((size_t)COLUMNS * shares_of(n, gates).groups * dim * 4, 256);
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
    Wide wide = wide_for(p->dim, p->type);
    for (const auto &a : all) {
        if (const int rc = check_rows(a.p, p->n, p->dim, a.stride, a.type, a.written)) return rc;
        wide.rows(a.p, a.stride, a.type);
    }
    wide.rows(p->gate, p->gate_stride, p->gate_type);
    for (const gdp_norm_params *s : {&p->post, &p->pre})
        if (s->form != GDP_NORM_NONE) wide.rows(s->weight, 0, s->type), wide.rows(s->bias, 0, s->type);
    if (!aligned(p->stats, 16)) return gdp_fail(GDP_E_BADARG, "gdp_norm: stats must be aligned to 16 bytes");
    const int64_t gates = p->gate ? p->gates : 0;
    const Shares shares = shares_of(p->n, gates);
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
    const int rc = p->n == 0 ? GDP_OK : with_types(p->type, p->stream_type, [&](auto T, auto S) {
        using TT = decltype(T);
        using SS = decltype(S);
        const auto run = [&](auto E) {
            return with_waves<E.value>(p->dim, [&](auto W, auto K, int threads) {
                return launch("gdp_norm_backward", norm_backward_kernel<TT, SS, W.value, K.value, E.value>, dim3((unsigned)shares.groups), threads, 0, queue, b,
                              static_cast<const typename SS::raw *>(p->stream), static_cast<const typename TT::raw *>(p->block), static_cast<const typename TT::raw *>(p->grad_normed),
                              static_cast<const typename SS::raw *>(p->grad_stream), static_cast<typename SS::raw *>(p->grad_residual), static_cast<typename TT::raw *>(p->grad_block));
            });
        };
        return wide.ok ? run(Int<TT::VEC>{}) : run(Int<1>{});
    });
    if (rc) return rc;
    const unsigned across = (unsigned)ceil_div(p->dim, (int64_t)ADD_COLUMNS);
    return count ? launch("gdp_norm_backward", norm_add_kernel, dim3(across, most, count), ADD_COLUMNS * ADD_ROWS, 0, queue, adds) : GDP_OK;
}
