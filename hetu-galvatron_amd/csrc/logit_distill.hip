// Distillation from a list of a teacher's most likely tokens: the divergence of each row of logits from it, and the gradient.
//
// Forward, one pass over the logits.  The listed tokens are marked in a bitmap in LDS (a bit for each column of the slice, looked at as one
// byte or half a byte for each read of 16 bytes) and left out of the sum of exponentials, so that what a teacher's rest is held against is
// the sum of the unlisted alone: 1 - sum(p) would have no digits left where a student is sure.  A listed token's own logit is read by
// itself.  With m and s of the unlisted and the list's logits everything else is a row's few numbers, which one wave takes in float64: 1 - sum(q) of
// float32 log probabilities keeps their digits only there, and 64 exponentials and logarithms are nothing next to a row.
//
// For any function of the probabilities p_b of the listed tokens and the rest, dL/dz_j = p_j (h_b - H), h_b = dL/dp_b of the alternative
// that j belongs to and H = sum of p_b h_b.  Of the unlisted this is one number for the row, C = p_rest (h_rest - H), times each one's share
// w_j = exp(scale (x_j - m_rest)) / s_rest of the unlisted: w_j and C stay in range where p_rest itself is far below float32.  So the
// gradient is elementwise with one exponential, and the listed places are written again.
//
// A row is one workgroup, or, where there are few rows, several of a slice each, whose sums a second kernel joins; the same kernel joins
// the shards of a vocabulary.
#include "ops_common.h"

#include <type_traits>

namespace {
using namespace ops;

constexpr int THREADS = 256;
constexpr int AHEAD = 4;                 // reads of 16 bytes in flight for each thread
constexpr int MOST_SLICES = 64;
constexpr int MOST_BITS = 1 << 18;       // columns of a slice: 32 KB of LDS
static_assert((int64_t)MOST_BITS * MOST_SLICES / 2 > GDP_MAX_VOCAB + 64, "slices go up to MOST_SLICES by factors of two");
static_assert(GDP_MAX_LISTED == 256, "four places for each lane of a wave");
constexpr int HEAD = 5;                  // numbers of stats in front of the places'
constexpr double LEAST_REST = 1.0 / (1 << 22);

// Largest logit of a part of a row and the sum of 2^(c (x - m)); -inf and 0 of nothing.
struct Sums {
    float m, s;
};
__device__ __forceinline__ Sums rescaled(Sums a, float m, float c)
{
    return {m, a.s == 0.0f ? 0.0f : a.s * exp2_fast(c * (finite_or_0(a.m) - finite_or_0(m)))};
}
__device__ __forceinline__ Sums wave_join(Sums a, float c)
{
    const float m = wave_max(a.m);
    return {m, wave_sum(rescaled(a, m, c).s)};
}
__device__ __forceinline__ double wave_sum(double v)   // in the same order for all lanes
{
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step);
    return v;
}

struct List {   // of each row, and its target
    const void *tokens, *targets;
    const float *teacher;
    int32_t listed, list_type, target_type;
};
struct Out {
    float *loss, *lse, *logp, *stats;
    float scale, beta;
    int32_t rest;
    int64_t whole;       // tokens outside [0, whole) are none
};
struct Part {   // of slices or shards: [parts][n][4], [parts][n][listed]
    float4 *sums;
    float *logits;
};

// The finish of a row, by one wave: PLACES places for each lane.  `all` of the unlisted; token (-1: none here), teacher and logit x of the
// places; x_target of the row's target.  LDS: `seen` and `probability` of GDP_MAX_LISTED each.
template <int PLACES>
__device__ void finish_row(const Out &o, const List &l, int64_t row, int lane, Sums all, const int32_t (&token)[PLACES], const float (&teacher)[PLACES],
                           const float (&x)[PLACES], float x_target, int32_t *seen, double *probability)
{
    constexpr double INF = __builtin_inf();
    const double scale = o.scale;
    double q[PLACES], lq[PLACES];   // of the token at a place, over all of its places
    bool counts[PLACES];            // the first place of a listed token
    float m = all.m;
    // without `rest` any scores will do: their largest is taken off first
    double level = 0.0;
    if (!o.rest) {
        float most = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < PLACES; ++j)
            if (token[j] >= 0) most = fmaxf(most, teacher[j]);
        level = finite_or_0(wave_max(most));
    }
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        const bool used = token[j] >= 0 && teacher[j] != -__builtin_inff();
        lq[j] = used ? (double)teacher[j] - level : -INF;
        q[j] = used ? exp(lq[j]) : 0.0;
        if (i < l.listed) {
            seen[i] = used ? token[j] : -1;
            probability[i] = q[j];
        }
        if (used) m = fmaxf(m, x[j]);
    }
    m = wave_max(m);
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
    bool is_listed[PLACES];
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        int first = GDP_MAX_LISTED, times = 0;
        double sum = 0.0;
        if (i < l.listed && token[j] >= 0)
            for (int k = 0; k < l.listed; ++k)
                if (seen[k] == token[j]) {
                    sum += probability[k];
                    first = first < k ? first : k;
                    ++times;
                }
        is_listed[j] = times > 0;
        counts[j] = first == i;
        // (the same bits at all places of a token, an unused one among them)
        if (times > 1)
            q[j] = sum, lq[j] = log(sum);
        else if (times == 1 && first != i)
            q[j] = sum, lq[j] = (double)l.teacher[row * l.listed + first] - level;
    }
    // probabilities of the student: of places, of the rest
    const float from = finite_or_0(m);
    const double d_out = ((double)finite_or_0(all.m) - from) * scale;
    double s = 0.0, d[PLACES];
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        d[j] = token[j] >= 0 ? ((double)x[j] - from) * scale : -INF;
        if (counts[j]) s += exp(d[j]);
    }
    const double s_out = all.s == 0.0f ? 0.0 : all.s * exp(d_out);
    s = wave_sum(s) + s_out;
    const bool nothing = s == 0.0;
    const double log_s = log(s), l_out = all.s == 0.0f ? -INF : d_out + log((double)all.s) - log_s, p_out = s_out / s;
    // of the teacher: over its list, of the rest
    double mass = 0.0;
#pragma unroll
    for (int j = 0; j < PLACES; ++j) mass += counts[j] ? q[j] : 0.0;
    mass = wave_sum(mass);
    double r = 0.0;
    if (o.rest) {
        r = 1.0 - mass;
        if (all.s == 0.0f) r = 0.0;
        else if (r < LEAST_REST) r = o.beta == 1.0f ? LEAST_REST : 0.0;
    } else {
        const double by = mass > 0.0 ? 1.0 / mass : mass == 0.0 ? 0.0 : mass, log_mass = mass == 0.0 ? 0.0 : log(mass);
#pragma unroll
        for (int j = 0; j < PLACES; ++j) q[j] *= by, lq[j] -= log_mass;
        mass = mass == 0.0 ? 0.0 : mass * by;
    }
    const double lr = log(r), beta = o.beta;
    double lp[PLACES], p[PLACES], a[PLACES];
    double loss = 0.0, mean = 0.0, a_out = 0.0, of_rest = 0.0;
#pragma unroll
    for (int j = 0; j < PLACES; ++j) lp[j] = d[j] - log_s, p[j] = exp(lp[j]);
    if (beta == 0.0) {
#pragma unroll
        for (int j = 0; j < PLACES; ++j)
            if (counts[j] && q[j] != 0.0) loss += q[j] * (lq[j] - lp[j]);
        loss = wave_sum(loss) + (r > 0.0 ? r * (lr - l_out) : 0.0);
        of_rest = (mass + r) * p_out - r;
    } else {
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            const double lm = beta == 1.0 ? lq[j] : log(beta * q[j] + (1.0 - beta) * p[j]);
            a[j] = p[j] == 0.0 ? 0.0 : lp[j] - lm;
            if (counts[j]) {
                mean += p[j] * a[j];
                if (beta != 1.0 && q[j] != 0.0) loss += q[j] * (lq[j] - lm);
            }
        }
        const double lm = beta == 1.0 ? lr : log(beta * r + (1.0 - beta) * p_out);
        a_out = p_out == 0.0 ? 0.0 : l_out - lm;
        mean = wave_sum(mean) + p_out * a_out;
        loss = wave_sum(loss) + (beta != 1.0 && r > 0.0 ? r * (lr - lm) : 0.0);
        loss = beta == 1.0 ? mean : beta * loss + (1.0 - beta) * mean;
        of_rest = (beta == 1.0 ? 1.0 : 1.0 - beta) * p_out * (a_out - mean);
    }
    const bool empty = nothing || (!o.rest && mass == 0.0 && s == s);   // no row, or no list
    if (s != s) loss = s;
    if (lane == 0) {
        o.loss[row] = empty ? 0.0f : (float)loss;
        o.lse[row] = nothing ? -__builtin_inff() : (float)(m * scale + log_s);
        if (l.targets) {
            const int64_t target = token_at(l.targets, l.target_type, row);
            const bool none = target < 0 || target >= o.whole;
            o.logp[row] = none ? 0.0f : nothing ? -__builtin_inff() : (float)(((double)x_target - m) * scale - log_s);
        }
    }
    if (!o.stats) return;
    float *const to = o.stats + row * (HEAD + l.listed);
    if (lane == 0) {
        to[0] = m, to[1] = (float)log_s;
        to[2] = all.m, to[3] = all.s == 0.0f ? -__builtin_inff() : logf(all.s);
        to[4] = empty || all.s == 0.0f ? 0.0f : (float)of_rest;
    }
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        double pull;
        if (!is_listed[j])
            pull = of_rest * exp((double)x[j] * scale - (double)finite_or_0(all.m) * scale - log((double)all.s));   // its share of the rest
        else if (beta == 0.0)
            pull = p[j] * (mass + r) - q[j];
        else
            pull = (beta == 1.0 ? 1.0 : 1.0 - beta) * p[j] * (a[j] - mean);
        if (i < l.listed) to[HEAD + i] = token[j] < 0 || empty || (!is_listed[j] && x[j] == -__builtin_inff()) ? 0.0f : (float)pull;
    }
}

struct Scan {
    int64_t n, vocab, stride, first;
    int32_t slices, width;   // vectors of a slice
    float c;
    List list;
    Out out;
    Part part;
};

template <typename T, int PLACES>
__global__ __launch_bounds__(THREADS) void distill_scan_kernel(Scan a, const typename T::raw *__restrict__ logits)
{
    constexpr int VEC = T::VEC, WAVES = THREADS / 64;
    extern __shared__ __align__(16) uint32_t bits[];   // a bit for each column of the slice's vectors
    __shared__ Sums of_wave[WAVES];
    __shared__ int32_t seen[64 * PLACES];
    __shared__ double probability[64 * PLACES];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t row = blockIdx.x / a.slices;
    const int slice = (int)(blockIdx.x % a.slices);
    const typename T::raw *const x = logits + row * a.stride;
    // Vectors are counted from the 16 bytes that the row begins in: the first and the last may be cut.
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(typename T::raw));
    const int vocab = (int)a.vocab, vectors = (vocab + off + VEC - 1) / VEC;
    const int v0 = slice * a.width, v1 = v0 + a.width < vectors ? v0 + a.width : vectors;
    const int from = v0 * VEC - off, to = v1 * VEC - off;   // columns of the slice, cut by the row's
    for (int i = t; i < (a.width * VEC + 31) / 32; i += THREADS) bits[i] = 0;
    int32_t token[PLACES];
    float teacher[PLACES], at_place[PLACES], of_target = -__builtin_inff();
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            const int i = lane + 64 * j;
            token[j] = -1, teacher[j] = at_place[j] = -__builtin_inff();
            if (i < a.list.listed) {
                const int64_t one = token_at(a.list.tokens, a.list.list_type, row * a.list.listed + i), local = one < 0 ? -1 : one - a.first;
                teacher[j] = a.list.teacher[row * a.list.listed + i];
                if (local >= 0 && local < vocab && local >= from && local < to) {
                    token[j] = (int32_t)local;
                    at_place[j] = T::up(x[local]);
                }
            }
        }
        if (lane == 0 && a.list.targets) {
            const int64_t target = token_at(a.list.targets, a.list.target_type, row), local = target < 0 ? -1 : target - a.first;
            if (local >= 0 && local < vocab && local >= from && local < to) of_target = T::up(x[local]);
        }
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < PLACES; ++j)
            if (token[j] >= 0 && teacher[j] != -__builtin_inff()) atomicOr(&bits[(token[j] - from) >> 5], 1u << ((token[j] - from) & 31));
    }
    __syncthreads();
    const float c = a.c;
    const uint8_t *const bytes = reinterpret_cast<const uint8_t *>(bits);
    Sums own{-__builtin_inff(), 0.0f};
    for (int base = v0; base < v1; base += THREADS * AHEAD) {
        Pack<T, VEC> p[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            if (v < v1 && j >= 0 && j + VEC <= vocab) {
                p[u].load(x + j);
            } else {
                float f[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = v < v1 && j + i >= 0 && j + i < vocab ? T::up(x[j + i]) : -__builtin_inff();
                p[u].set(f);
            }
        }
        float most = own.m;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t - v0;
            if (v < v1 - v0) {
                const uint32_t out = VEC == 8 ? bytes[v] : (bytes[v >> 1] >> (4 * (v & 1))) & 15u;
                if (out) {
                    float f[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f[i] = out >> i & 1 ? -__builtin_inff() : p[u][i];
                    p[u].set(f);
                }
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) most = fmaxf(most, p[u][i]);
        }
        own = rescaled(own, most, c);
        const float level = finite_or_0(most);   // (subtracted first: a row may hold a type's lowest value alone)
        float sum = 0.0f;                        // of these reads: a row's sums then are of few terms each
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum += exp2_fast((p[u][i] - level) * c);
        own.s += sum;
    }
    own = wave_join(own, c);
    if (lane == 0) of_wave[wave] = own;
    __syncthreads();
    if (wave != 0) return;
    float m = of_wave[0].m;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, of_wave[w].m);
    Sums all{m, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all.s += rescaled(of_wave[w], m, c).s;
    if (!a.part.sums) {
        finish_row<PLACES>(a.out, a.list, row, lane, all, token, teacher, at_place, of_target, seen, probability);
        return;
    }
    const int64_t at = (int64_t)slice * a.n + row;
    if (lane == 0) a.part.sums[at] = make_float4(all.m, all.s, of_target, 0.0f);
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        if (i < a.list.listed) a.part.logits[at * a.list.listed + i] = at_place[j];
    }
}

struct Join {
    int64_t n;
    int32_t parts;
    float c;
    List list;
    Part in;
    Out out;
    Part part;   // written instead of out where its sums are not null: slices of a shard
};

// The larger; NaN where one of them is.
__device__ __forceinline__ float most_or_nan(float a, float b) { return a > b || a != a ? a : b; }

// A wave for each row.
template <int PLACES> __global__ __launch_bounds__(64) void distill_join_kernel(Join a)
{
    __shared__ int32_t seen[64 * PLACES];
    __shared__ double probability[64 * PLACES];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int listed = a.list.listed;
    Sums own{-__builtin_inff(), 0.0f};
    float of_target = -__builtin_inff();
    if (lane < a.parts) {
        const float4 s = a.in.sums[(int64_t)lane * a.n + row];
        own = {s.x, s.y};
        of_target = s.z;
    }
    int32_t token[PLACES];
    float teacher[PLACES], x[PLACES];
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        token[j] = -1, teacher[j] = x[j] = -__builtin_inff();
        if (i < listed) {
            const int64_t one = token_at(a.list.tokens, a.list.list_type, row * listed + i);
            if (one >= 0 && one < a.out.whole) token[j] = (int32_t)one;
            teacher[j] = a.list.teacher[row * listed + i];
#pragma unroll 4
            for (int p = 0; p < a.parts; ++p) x[j] = most_or_nan(a.in.logits[((int64_t)p * a.n + row) * listed + i], x[j]);
        }
    }
    const Sums all = wave_join(own, a.c);
    const bool no_number = __ballot(of_target != of_target) != 0;
    of_target = no_number ? __builtin_nanf("") : wave_max(of_target);
    if (!a.part.sums) {
        finish_row<PLACES>(a.out, a.list, row, lane, all, token, teacher, x, of_target, seen, probability);
        return;
    }
    if (lane == 0) a.part.sums[row] = make_float4(all.m, all.s, of_target, 0.0f);
#pragma unroll
    for (int j = 0; j < PLACES; ++j)
        if (lane + 64 * j < listed) a.part.logits[row * listed + lane + 64 * j] = x[j];
}

struct Grad {
    int64_t vocab, stride, out_stride, first, whole;
    int32_t slices, width;
    float scale;
    List list;
    const float *stats, *grad_loss, *grad_lse, *grad_logp;
};

template <typename T>
__global__ __launch_bounds__(THREADS) void distill_grad_kernel(Grad a, const typename T::raw *logits, typename T::raw *out)
{
    constexpr int VEC = T::VEC, ENTRIES = (GDP_MAX_LISTED + 1 + THREADS - 1) / THREADS;
    __shared__ int32_t target_is_listed;
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x / a.slices;
    const int slice = (int)(blockIdx.x % a.slices);
    const typename T::raw *const x = logits + row * a.stride;
    typename T::raw *const y = out + row * a.out_stride;
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(typename T::raw));
    const int vocab = (int)a.vocab, vectors = (vocab + off + VEC - 1) / VEC;
    const int v0 = slice * a.width, v1 = v0 + a.width < vectors ? v0 + a.width : vectors;
    const int from = v0 * VEC - off, to = v1 * VEC - off;
    const int listed = a.list.listed;
    const float *const stats = a.stats + row * (HEAD + listed);
    const float m = stats[0], log_s = stats[1], m_out = stats[2], log_out = stats[3];
    const bool dead = log_s < -__FLT_MAX__, none = log_out < -__FLT_MAX__;   // no logit above -inf; none that is not listed
    int64_t target = a.list.targets && a.grad_logp ? token_at(a.list.targets, a.list.target_type, row) : -1;
    if (target >= a.whole) target = -1;
    const float g = target >= 0 && !dead ? a.grad_logp[row] : 0.0f;
    const float of_p = dead ? 0.0f : (a.grad_lse ? a.grad_lse[row] : 0.0f) - g, of_loss = a.grad_loss ? a.grad_loss[row] : 0.0f;
    const auto p_of = [&](float f) { return dead ? 0.0f : exp2_fast(fmaf(f - m, a.scale, -log_s) * LOG2E); };
    // w_j: the share of the unlisted; p_j of them is w_j times p_rest
    const float p_out = none ? 0.0f : exp2_fast((fmaf(m_out - m, a.scale, log_out) - log_s) * LOG2E);
    const float factor = none ? 0.0f : a.scale * ((of_loss != 0.0f ? of_loss * stats[4] : 0.0f) + (of_p != 0.0f ? of_p * p_out : 0.0f));
    const float level = none ? 0.0f : m_out, away = none ? __builtin_inff() : log_out;
    const auto grad_of = [&](float f) { return factor * exp2_fast(fmaf(f - level, a.scale, -away) * LOG2E); };
    // The listed places and the target, from their logits, before anything is written (out may be the logits).  A token in several
    // places has the same gradient at each.
    if (t == 0) target_is_listed = 0;
    __syncthreads();
    int32_t column[ENTRIES];
    float value[ENTRIES];
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k) {
        const int e = t + k * THREADS;
        column[k] = -1;
        if (e < listed) {
            const int64_t one = token_at(a.list.tokens, a.list.list_type, row * listed + e), local = one < 0 ? -1 : one - a.first;
            if (local >= 0 && local < vocab && local >= from && local < to) {
                column[k] = (int32_t)local;
                value[k] = of_loss != 0.0f ? of_loss * stats[HEAD + e] : 0.0f;
                if (of_p != 0.0f) value[k] += of_p * p_of(T::up(x[local]));
                if (one == target) value[k] += g, target_is_listed = 1;
                value[k] *= a.scale;
            }
        }
    }
    __syncthreads();
    float again = 0.0f;
    int32_t at_target = -1;
    if (t == 0 && target >= 0 && !target_is_listed) {
        const int64_t local = target - a.first;
        if (local >= 0 && local < vocab && local >= from && local < to) {
            at_target = (int32_t)local;
            again = grad_of(T::up(x[local])) + a.scale * g;
        }
    }
    __syncthreads();
    for (int base = v0; base < v1; base += THREADS * AHEAD) {
        Pack<T, VEC> p[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            if (v < v1 && j >= 0 && j + VEC <= vocab) p[u].load(x + j);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            if (v >= v1) continue;
            if (j >= 0 && j + VEC <= vocab) {
                float f[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = grad_of(p[u][i]);
                p[u].set(f);
                p[u].store(y + j);
            } else {
                for (int i = 0; i < VEC; ++i)
                    if (j + i >= 0 && j + i < vocab) y[j + i] = T::down(grad_of(T::up(x[j + i])));
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k)
        if (column[k] >= 0) y[column[k]] = T::down(value[k]);
    if (at_target >= 0) y[at_target] = T::down(again);
}

// ---- host ----
// How a row is shared out: slices of 512 vectors (8 KB) at least, 1024 workgroups, and no more columns in a slice than LDS has bits for.
struct Split {
    int slices, width;
};
Split split_of(int64_t n, int64_t vocab, int type)
{
    const int vec = 16 / size_of(type);
    const int64_t vectors = ceil_div(vocab, (int64_t)vec) + 1;   // one more where a row begins within 16 bytes
    int64_t slices = 1;
    while (slices < MOST_SLICES && n * slices < 1024 && vectors / (slices * 2) >= 512) slices *= 2;
    while (slices < MOST_SLICES && ceil_div(vectors, slices) * vec > MOST_BITS) slices *= 2;
    const int64_t width = ceil_div(vectors, slices);
    return {(int)ceil_div(vectors, width), (int)width};
}
size_t sums_bytes(int64_t parts, int64_t n) { return round_up((size_t)parts * n * 16, 256); }
size_t part_bytes(int64_t parts, int64_t n, int listed) { return sums_bytes(parts, n) + round_up((size_t)parts * n * listed * 4, 256); }
Part part_at(void *p, int64_t parts, int64_t n)
{
    return {static_cast<float4 *>(p), reinterpret_cast<float *>(static_cast<char *>(p) + sums_bytes(parts, n))};
}

constexpr int64_t MOST_ROWS = (int64_t)1 << 21, MOST_GROUPS = (int64_t)1 << 23;   // a grid has less than 2^32 threads
int check(int64_t n, int64_t vocab, int64_t first, int type, int listed)
{
    if (n < 0 || vocab < 1 || first < 0) return gdp_fail(GDP_E_BADARG, "gdp_distill: a size is negative, or there are no columns");
    if (n > MOST_ROWS || vocab > GDP_MAX_VOCAB || first > INT32_MAX - vocab)
        return gdp_fail(GDP_E_BADARG, "gdp_distill: more than 2^21 rows or GDP_MAX_VOCAB columns, or a token above 2^31");
    if (!type_ok(type)) return gdp_fail(GDP_E_BADARG, "gdp_distill: unknown element type");
    if (listed < 1 || listed > GDP_MAX_LISTED) return gdp_fail(GDP_E_BADARG, "gdp_distill: listed must be 1 to GDP_MAX_LISTED");
    return GDP_OK;
}
int check_list(const List &l)
{
    if (!token_type_ok(l.list_type) || (l.targets && !token_type_ok(l.target_type))) return gdp_fail(GDP_E_BADARG, "gdp_distill: unknown token type");
    if (!l.tokens || !l.teacher) return gdp_fail(GDP_E_BADARG, "gdp_distill: null pointer");
    if (!aligned(l.tokens, l.list_type == GDP_I64 ? 8 : 4) || !aligned(l.teacher, 4) || !aligned(l.targets, l.target_type == GDP_I64 ? 8 : 4))
        return gdp_fail(GDP_E_BADARG, "gdp_distill: a pointer is not aligned to its elements");
    return GDP_OK;
}
int check_scale(float scale)
{
    return scale > 0.0f && scale < 1e30f ? GDP_OK : gdp_fail(GDP_E_BADARG, "gdp_distill: scale must be positive and below 1e30");
}
int check_form(float beta, int rest)
{
    if (!(beta >= 0.0f && beta <= 1.0f)) return gdp_fail(GDP_E_BADARG, "gdp_distill: beta must be 0 to 1");
    return beta == 1.0f && !rest ? gdp_fail(GDP_E_BADARG, "gdp_distill: beta 1 needs the rest") : GDP_OK;
}
int check_logits(const void *p, int64_t n, int64_t vocab, int64_t stride, int type, bool written)
{
    if (!p) return gdp_fail(GDP_E_BADARG, "gdp_distill: null pointer");
    if (!rows_ok(n, vocab, stride, written)) return gdp_fail(GDP_E_BADARG, "gdp_distill: a row stride is negative, too large, or below the width of rows that are written");
    return aligned(p, size_of(type)) ? GDP_OK : gdp_fail(GDP_E_BADARG, "gdp_distill: a pointer is not aligned to its elements");
}
int check_out(const Out &o, const List &l)
{
    if (!o.loss || !o.lse || !l.targets != !o.logp) return gdp_fail(GDP_E_BADARG, "gdp_distill: null pointer, or one of targets and logp alone");
    return aligned(o.loss, 4) && aligned(o.lse, 4) && aligned(o.logp, 4) && aligned(o.stats, 4) ? GDP_OK
                                                                                              : gdp_fail(GDP_E_BADARG, "gdp_distill: a pointer is not aligned to its elements");
}

int scan(Scan s, const void *logits, int type, const Split &split, const char *who, void *stream)
{
    s.slices = split.slices, s.width = split.width;
    return with_type(type, [&](auto T) {
        using TT = decltype(T);
        const auto *x = static_cast<const typename TT::raw *>(logits);
        const dim3 grid((unsigned)(s.n * split.slices));
        const size_t lds = round_up(ceil_div((size_t)split.width * TT::VEC, (size_t)32) * 4, 16);
        return s.list.listed <= 64 ? launch(who, distill_scan_kernel<TT, 1>, grid, THREADS, lds, stream, s, x)
                                   : launch(who, distill_scan_kernel<TT, 4>, grid, THREADS, lds, stream, s, x);
    });
}
int join(const Join &j, const char *who, void *stream)
{
    const dim3 grid((unsigned)j.n);
    return j.list.listed <= 64 ? launch(who, distill_join_kernel<1>, grid, 64, 0, stream, j) : launch(who, distill_join_kernel<4>, grid, 64, 0, stream, j);
}
// Slices of a row, joined where there are several.
int rows(Scan s, const void *logits, int type, void *workspace, size_t bytes, const char *who, void *stream)
{
    const Split split = split_of(s.n, s.vocab, type);
    if (s.n * split.slices > MOST_GROUPS) return gdp_fail(GDP_E_BADARG, "gdp_distill: too many rows of so many columns");
    if (split.slices == 1) return scan(s, logits, type, split, who, stream);
    if (!workspace || !aligned(workspace, 256) || bytes < part_bytes(split.slices, s.n, s.list.listed))
        return gdp_fail(GDP_E_BADARG, "gdp_distill: the workspace is smaller than gdp_distill_workspace says, or not aligned to 256 bytes");
    Join j{s.n, split.slices, s.c, s.list, part_at(workspace, split.slices, s.n), s.out, s.part};
    s.part = j.in;
    if (const int rc = scan(s, logits, type, split, who, stream)) return rc;
    return join(j, who, stream);
}

}  // namespace

extern "C" int gdp_distill_workspace(int64_t n, int64_t vocab, int32_t logits_type, int32_t listed, size_t *bytes)
{
    gdp_clear_error();
    if (!bytes) return gdp_fail(GDP_E_BADARG, "gdp_distill: null argument");
    if (const int rc = check(n, vocab, 0, logits_type, listed)) return rc;
    const Split s = split_of(n, vocab, logits_type);
    *bytes = s.slices > 1 ? part_bytes(s.slices, n, listed) : 0;
    return GDP_OK;
}

extern "C" int gdp_distill_forward(const gdp_distill *d, void *stream)
{
    gdp_clear_error();
    if (!d) return gdp_fail(GDP_E_BADARG, "gdp_distill: null argument");
    if (const int rc = check(d->n, d->vocab, 0, d->logits_type, d->listed)) return rc;
    if (const int rc = check_scale(d->scale)) return rc;
    if (const int rc = check_form(d->beta, d->rest)) return rc;
    if (d->n == 0) return GDP_OK;
    const List list{d->tokens, d->targets, d->teacher, d->listed, d->list_type, d->target_type};
    const Out out{d->loss, d->lse, d->logp, d->stats, d->scale, d->beta, d->rest, d->vocab};
    if (const int rc = check_list(list)) return rc;
    if (const int rc = check_out(out, list)) return rc;
    if (const int rc = check_logits(d->logits, d->n, d->vocab, d->logits_stride, d->logits_type, false)) return rc;
    return rows({d->n, d->vocab, d->logits_stride, 0, 0, 0, d->scale * LOG2E, list, out, {}}, d->logits, d->logits_type, d->workspace, d->workspace_bytes,
                "gdp_distill_forward", stream);
}

extern "C" int gdp_distill_parts(const gdp_distill_part *d, void *stream)
{
    gdp_clear_error();
    if (!d) return gdp_fail(GDP_E_BADARG, "gdp_distill: null argument");
    if (const int rc = check(d->n, d->vocab, d->first, d->logits_type, d->listed)) return rc;
    if (const int rc = check_scale(d->scale)) return rc;
    if (d->n == 0) return GDP_OK;
    const List list{d->tokens, d->targets, d->teacher, d->listed, d->list_type, d->target_type};
    if (const int rc = check_list(list)) return rc;
    if (!d->sums || !aligned(d->sums, 16) || !d->listed_logits || !aligned(d->listed_logits, 4))
        return gdp_fail(GDP_E_BADARG, "gdp_distill: null pointer, or sums not aligned to 16 bytes");
    if (const int rc = check_logits(d->logits, d->n, d->vocab, d->logits_stride, d->logits_type, false)) return rc;
    Out out{};
    out.whole = INT32_MAX;
    return rows({d->n, d->vocab, d->logits_stride, d->first, 0, 0, d->scale * LOG2E, list, out, {reinterpret_cast<float4 *>(d->sums), d->listed_logits}}, d->logits,
                d->logits_type, d->workspace, d->workspace_bytes, "gdp_distill_parts", stream);
}

extern "C" int gdp_distill_join(const gdp_distill_joint *d, void *stream)
{
    gdp_clear_error();
    if (!d) return gdp_fail(GDP_E_BADARG, "gdp_distill: null argument");
    if (d->n < 0 || d->n > MOST_ROWS || d->vocab < 1 || d->vocab > INT32_MAX) return gdp_fail(GDP_E_BADARG, "gdp_distill: a size is out of range");
    if (d->parts < 1 || d->parts > GDP_MAX_LOGPROB_PARTS) return gdp_fail(GDP_E_BADARG, "gdp_distill: parts must be 1 to GDP_MAX_LOGPROB_PARTS");
    if (d->listed < 1 || d->listed > GDP_MAX_LISTED) return gdp_fail(GDP_E_BADARG, "gdp_distill: listed must be 1 to GDP_MAX_LISTED");
    if (const int rc = check_scale(d->scale)) return rc;
    if (const int rc = check_form(d->beta, d->rest)) return rc;
    if (d->n == 0) return GDP_OK;
    const List list{d->tokens, d->targets, d->teacher, d->listed, d->list_type, d->target_type};
    const Out out{d->loss, d->lse, d->logp, d->stats, d->scale, d->beta, d->rest, d->vocab};
    if (const int rc = check_list(list)) return rc;
    if (const int rc = check_out(out, list)) return rc;
    if (!d->sums || !aligned(d->sums, 16) || !d->listed_logits || !aligned(d->listed_logits, 4))
        return gdp_fail(GDP_E_BADARG, "gdp_distill: null pointer, or sums not aligned to 16 bytes");
    const Part in{reinterpret_cast<float4 *>(const_cast<float *>(d->sums)), const_cast<float *>(d->listed_logits)};
    return join({d->n, d->parts, d->scale * LOG2E, list, in, out, {}}, "gdp_distill_join", stream);
}

extern "C" int gdp_distill_backward(const gdp_distill_grad *d, void *stream)
{
    gdp_clear_error();
    if (!d) return gdp_fail(GDP_E_BADARG, "gdp_distill: null argument");
    if (const int rc = check(d->n, d->vocab, d->first, d->logits_type, d->listed)) return rc;
    if (d->whole_vocab < 1) return gdp_fail(GDP_E_BADARG, "gdp_distill: a size is out of range");
    if (const int rc = check_scale(d->scale)) return rc;
    if (d->n == 0) return GDP_OK;
    const List list{d->tokens, d->targets, d->stats, d->listed, d->list_type, d->target_type};   // (no place's log probability is needed)
    if (const int rc = check_list(list)) return rc;
    if (const int rc = check_logits(d->logits, d->n, d->vocab, d->logits_stride, d->logits_type, false)) return rc;
    if (const int rc = check_logits(d->out, d->n, d->vocab, d->out_stride, d->logits_type, true)) return rc;
    if (d->grad_logp && !d->targets) return gdp_fail(GDP_E_BADARG, "gdp_distill: a gradient of logp without targets");
    if (!aligned(d->grad_loss, 4) || !aligned(d->grad_lse, 4) || !aligned(d->grad_logp, 4)) return gdp_fail(GDP_E_BADARG, "gdp_distill: a pointer is not aligned to its elements");
    if (d->out == d->logits && d->n > 1 && d->out_stride != d->logits_stride) return gdp_fail(GDP_E_BADARG, "gdp_distill: a gradient in the place of the logits needs their stride");
    const int vec = 16 / size_of(d->logits_type);
    const int64_t vectors = ceil_div(d->vocab, (int64_t)vec) + 1;
    int64_t slices = 1;   // two rounds of reads for each workgroup, more where the grid would be too large
    while (vectors / slices > 2 * THREADS * AHEAD && d->n * slices < (1 << 22)) slices *= 2;
    const int64_t width = ceil_div(vectors, slices);
    slices = ceil_div(vectors, width);
    const Grad g{d->vocab, d->logits_stride, d->out_stride, d->first, d->whole_vocab, (int32_t)slices, (int32_t)width, d->scale, list, d->stats,
                 d->grad_loss, d->grad_lse, d->grad_logp};
    return with_type(d->logits_type, [&](auto T) {
        using TT = decltype(T);
        return launch("gdp_distill_backward", distill_grad_kernel<TT>, dim3((unsigned)(d->n * slices)), THREADS, 0, stream, g,
                      static_cast<const typename TT::raw *>(d->logits), static_cast<typename TT::raw *>(d->out));
    });
}
