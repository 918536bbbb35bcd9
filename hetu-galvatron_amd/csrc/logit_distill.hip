// Distillation from a list of a teacher's most likely tokens: the divergence of each row of logits from it, and the gradient.
//
// Forward, one pass over the logits.  The listed tokens are marked in a bitmap in LDS (a bit for each column of the slice, looked at as one
// byte or half a byte for each read of 16 bytes) and left out of the sum of exponentials, so that what a teacher's rest is held against is
// the sum of the unlisted alone: 1 - sum(p) would have no digits left where a student is sure.  A listed token's own logit is read by
// itself.  With m and s of the unlisted and the list's logits everything else is a row's few numbers, which one wave takes in float64: 1 - sum(q) of
// float32 log probabilities keeps their digits only there.  That is 3 us of a wave, behind long rows hidden, of short ones the larger part.
//
// For any function of the probabilities p_b of the listed tokens and the rest, dL/dz_j = p_j (h_b - H), h_b = dL/dp_b of the alternative
// that j belongs to and H = sum of p_b h_b.  Of the unlisted this is one number for the row, C = p_rest (h_rest - H), times each one's share
// w_j = exp(scale (x_j - m_rest)) / s_rest of the unlisted: w_j and C stay in range where p_rest itself is far below float32.  So the
// gradient is elementwise with one exponential, and the listed places are written again.
//
// A row is one workgroup, or a wave of its own where rows are short and many, or, where there are few rows, several workgroups of a slice
// each, whose sums a second kernel joins; the same kernel joins the shards of a vocabulary.
#include "ops_common.h"

#include <type_traits>

namespace {
using namespace ops;

constexpr int THREADS = 256;
constexpr int AHEAD = 2;                 // reads of 16 bytes in flight for each thread
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
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ double plus_moved(double v)   // + 0 where there is no source
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t moved = (uint64_t)dpp<CTRL, ROWS>((uint32_t)(b >> 32), 0u) << 32 | dpp<CTRL, ROWS>((uint32_t)b, 0u);
    return v + __builtin_bit_cast(double, moved);
}
__device__ __forceinline__ double of_lane(double v, int lane)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t there = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)b, lane);
    return __builtin_bit_cast(double, there);
}
__device__ __forceinline__ double wave_sum(double v)
{
    v = plus_moved<ROW_SHR1>(v);
    v = plus_moved<ROW_SHR2>(v);
    v = plus_moved<ROW_SHR4>(v);
    v = plus_moved<ROW_SHR8>(v);
    v = plus_moved<BCAST15, 0xa>(v);
    v = plus_moved<BCAST31, 0xc>(v);
    return of_lane(v, 63);
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
struct Part {   // of slices or shards: [parts][n][4]; of shards [parts][n][listed], of slices one for all, of which each writes its own tokens'
    float4 *sums;
    float *logits;
};

// The finish of a row, by one wave: PLACES places for each lane.  `all` of the unlisted; token (-1: none here), teacher and logit x of the
// places; x_target of the row's target; whether tokens may be there at several places.  LDS: `seen` and `probability` of 64 PLACES each.
// Some 8 exponentials and logarithms of float64: 3 us a wave, hidden behind other rows' reads where there are many.
template <int PLACES>
__device__ void finish_row(const Out &o, const List &l, int64_t row, int lane, Sums all, const int32_t (&token)[PLACES], const float (&teacher)[PLACES],
                           const float (&x)[PLACES], float x_target, bool repeats, int32_t *seen, double *probability)
{
    constexpr double INF = __builtin_inf();
    const double scale = o.scale;
    double q[PLACES], lq[PLACES];   // of the token at a place, over all of its places
    bool is_listed[PLACES];         // ... is at a place that is used
    bool counts[PLACES];            // the first of these
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
        counts[j] = is_listed[j] = token[j] >= 0 && teacher[j] != -__builtin_inff();
        lq[j] = !counts[j] ? -INF : teacher[j] == __builtin_inff() ? __builtin_nan("") : (double)teacher[j] - level;
        q[j] = exp(lq[j]);
        if (counts[j]) m = fmaxf(m, x[j]);
    }
    m = wave_max(m);
    if (repeats) {
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            seen[lane + 64 * j] = counts[j] ? token[j] : -1;
            probability[lane + 64 * j] = q[j];
        }
        __builtin_amdgcn_wave_barrier();
        __threadfence_block();
        int first[PLACES], times[PLACES];
        double sum[PLACES];
#pragma unroll
        for (int j = 0; j < PLACES; ++j) first[j] = lane + 64 * j, times[j] = 0, sum[j] = 0.0;
        for (int k = 0; k < l.listed; ++k) {
            const int one = seen[k];
#pragma unroll
            for (int j = 0; j < PLACES; ++j)
                if (one >= 0 && one == token[j]) {
                    sum[j] += probability[k];
                    first[j] = times[j]++ ? first[j] : k;
                }
        }
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            is_listed[j] = times[j] > 0;
            counts[j] = times[j] > 0 && first[j] == lane + 64 * j;
            // (the same bits at all places of a token, an unused one among them)
            if (times[j] > 1) {
                q[j] = sum[j], lq[j] = log(sum[j]);
                if (sum[j] < __DBL_MIN__) {   // (what float64 has few digits for, or none: relative to the token's largest)
                    const float *const of_row = l.teacher + row * l.listed;
                    float most = -__builtin_inff();
                    for (int k = 0; k < l.listed; ++k)
                        if (seen[k] == token[j]) most = fmaxf(most, of_row[k]);
                    double relative = 0.0;
                    for (int k = 0; k < l.listed; ++k)
                        if (seen[k] == token[j]) relative += exp((double)of_row[k] - most);
                    lq[j] = (double)most - level + log(relative);
                }
            } else if (times[j] == 1 && !counts[j])
                q[j] = sum[j], lq[j] = (double)l.teacher[row * l.listed + first[j]] - level;
        }
    }
    // probabilities of the student, relative to its largest logit: of places, of the rest
    const float from = finite_or_0(m);
    const double d_out = ((double)finite_or_0(all.m) - from) * scale, s_out = all.s == 0.0f ? 0.0 : all.s * exp(d_out);
    double s = 0.0, mass = 0.0, lp[PLACES], p[PLACES];
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        lp[j] = token[j] >= 0 ? ((double)x[j] - from) * scale : -INF;
        p[j] = exp(lp[j]);
        s += counts[j] ? p[j] : 0.0;
        mass += counts[j] ? q[j] : 0.0;
    }
    s = wave_sum(s) + s_out;
    mass = wave_sum(mass);
    // of the teacher: its rest, or its list normed
    double r = 0.0, norm = 1.0;
    if (o.rest) {
        r = all.s == 0.0f ? 0.0 : 1.0 - mass;
        if (all.s != 0.0f && r < LEAST_REST) r = o.beta == 1.0f ? LEAST_REST : 0.0;
    } else if (mass != 0.0)
        norm = mass;
    // the logarithms of four numbers, a lane for each
    const double logs = log(lane == 0 ? s : lane == 1 ? (double)all.s : lane == 2 ? norm : r);
    const double log_s = of_lane(logs, 0), log_out = of_lane(logs, 1), log_norm = of_lane(logs, 2), lr = of_lane(logs, 3);
    const bool nothing = s == 0.0;
    // (a teacher that is no number makes the student's probabilities none, and so the loss and all that goes by it)
    const double l_out = all.s == 0.0f ? -INF : d_out + log_out - log_s, of_s = mass != mass ? mass : 1.0 / s, p_out = s_out * of_s, of_norm = 1.0 / norm;
    mass *= of_norm;
#pragma unroll
    for (int j = 0; j < PLACES; ++j) q[j] *= of_norm, lq[j] -= log_norm, lp[j] -= log_s, p[j] *= of_s;
    const double beta = o.beta;
    double loss = 0.0, mean = 0.0, of_rest, pull[PLACES];
    if (beta == 0.0) {
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            if (counts[j] && q[j] != 0.0) loss += q[j] * (lq[j] - lp[j]);
            pull[j] = p[j] * (mass + r) - q[j];
        }
        loss = wave_sum(loss) + (r > 0.0 ? r * (lr - l_out) : 0.0);
        of_rest = (mass + r) * p_out - r;
    } else {
        const bool between = beta != 1.0;
        const double of_p = between ? 1.0 - beta : 1.0;
        double a[PLACES];   // ln p less that of what it is held against
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            const double lm = between ? log(beta * q[j] + of_p * p[j]) : lq[j];
            a[j] = p[j] == 0.0 ? 0.0 : lp[j] - lm;
            if (counts[j]) {
                mean += p[j] * a[j];
                if (between && q[j] != 0.0) loss += q[j] * (lq[j] - lm);
            }
        }
        const double lm = between ? log(beta * r + of_p * p_out) : lr, a_out = p_out == 0.0 ? 0.0 : l_out - lm;
        mean = wave_sum(mean) + p_out * a_out;
        if (between) loss = wave_sum(loss) + (r > 0.0 ? r * (lr - lm) : 0.0);
        loss = between ? beta * loss + of_p * mean : mean;
        of_rest = of_p * p_out * (a_out - mean);
#pragma unroll
        for (int j = 0; j < PLACES; ++j) pull[j] = of_p * p[j] * (a[j] - mean);
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
        to[2] = all.m, to[3] = (float)log_out;
        to[4] = empty || all.s == 0.0f ? 0.0f : (float)of_rest;
    }
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        if (i >= l.listed) continue;
        const bool of_others = token[j] >= 0 && !is_listed[j];   // a token at places that are not used: its share of the rest
        if (of_others) pull[j] = x[j] == -__builtin_inff() ? 0.0 : of_rest * exp(((double)x[j] - all.m) * scale - log_out);
        to[HEAD + i] = token[j] < 0 || empty ? 0.0f : (float)pull[j];
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

// Bound by memory where rows are long and many: 8192 x 128256 bf16 with 20 listed tokens 320 us, 2.1 GB at 6.6 TB/s; 2048 x 50257 float16 with 64 and beta
// 0.5 48 us, 4.3 TB/s: two rounds of workgroups, and a finish of 3 us behind each row.  Rows of 2 KB are mostly finish: 32089 x 1180 57 us, some 25 less without it.
// Few rows wait for memory four times (lists, bitmap, logits, the join): 16 x 128256 9 us.
// PLACES: of each lane of the wave that finishes, 1 or 4; the finish of four holds 100 registers.  FINISH: whole rows are finished here.  PAST: read past the caches.
template <typename T, int PLACES, bool FINISH, bool PAST, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void distill_scan_kernel(Scan a, const typename T::raw *__restrict__ logits)
{
    constexpr int VEC = T::VEC, THREADS = 64 * WAVES;
    extern __shared__ __align__(16) uint32_t bits[];   // a bit for each column of the slice's vectors
    __shared__ Sums of_wave[WAVES];
    __shared__ int32_t seen[64 * PLACES], repeats;
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
    Pack<T, VEC> p[AHEAD];
    const auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            if (v < v1 && j >= 0 && j + VEC <= vocab) {
                if constexpr (PAST)
                    p[u].load_past(x + j);
                else
                    p[u].load(x + j);
            } else {
                float f[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = v < v1 && j + i >= 0 && j + i < vocab ? T::up(x[j + i]) : -__builtin_inff();
                p[u].set(f);
            }
        }
    };
    int32_t token[PLACES];
    float teacher[PLACES];
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            const int i = lane + 64 * j;
            token[j] = -1, teacher[j] = -__builtin_inff();
            if (i < a.list.listed) {
                const int64_t one = token_at(a.list.tokens, a.list.list_type, row * a.list.listed + i), local = one < 0 || one >= a.out.whole ? -1 : one - a.first;
                teacher[j] = a.list.teacher[row * a.list.listed + i];
                if (local >= 0 && local < vocab && local >= from && local < to) token[j] = (int32_t)local;
            }
        }
    }
    load(v0);   // (on their way while the bitmap is made)
    for (int i = t; i < (a.width * VEC + 31) / 32; i += THREADS) bits[i] = 0;
    if (t == 0) repeats = 0;
    __syncthreads();
    typename T::raw at_place[PLACES], of_target = T::down(-__builtin_inff());
    if (wave == 0) {
        bool again = false;
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            const uint32_t bit = 1u << ((token[j] - from) & 31);
            if (token[j] >= 0 && teacher[j] != -__builtin_inff()) again |= (atomicOr(&bits[(token[j] - from) >> 5], bit) & bit) != 0;
        }
#pragma unroll
        for (int j = 0; j < PLACES; ++j) {
            at_place[j] = T::down(-__builtin_inff());
            if (token[j] < 0) continue;
            at_place[j] = x[token[j]];
            again |= teacher[j] == -__builtin_inff() && (bits[(token[j] - from) >> 5] >> ((token[j] - from) & 31) & 1);
        }
        if (again) repeats = 1;
        if (lane == 0 && a.list.targets) {
            const int64_t target = token_at(a.list.targets, a.list.target_type, row), local = target < 0 ? -1 : target - a.first;
            if (local >= 0 && local < vocab && local >= from && local < to) of_target = x[local];
        }
    }
    __syncthreads();
    const float c = a.c;
    const uint8_t *const bytes = reinterpret_cast<const uint8_t *>(bits);
    Sums own{-__builtin_inff(), 0.0f};
    for (int base = v0; base < v1; base += THREADS * AHEAD) {
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
        if (base + THREADS * AHEAD < v1) load(base + THREADS * AHEAD);
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
    float x_k[PLACES];
#pragma unroll
    for (int j = 0; j < PLACES; ++j) x_k[j] = T::up(at_place[j]);
    if constexpr (FINISH)
        if (!a.part.sums) {
            finish_row<PLACES>(a.out, a.list, row, lane, all, token, teacher, x_k, T::up(of_target), repeats != 0, seen, probability);
            return;
        }
    const int64_t at = (int64_t)slice * a.n + row;
    if (lane == 0) a.part.sums[at] = make_float4(all.m, all.s, T::up(of_target), repeats ? 1.0f : 0.0f);
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        if (i < a.list.listed && (a.slices == 1 || token[j] >= 0)) a.part.logits[row * a.list.listed + i] = x_k[j];
    }
}

struct Join {
    int64_t n;
    int64_t first, columns;  // the tokens that the lists are of (none where columns is not above 0)
    int32_t parts, lists;    // lists: 1 of slices
    float c;
    List list;
    Part in;
    Out out;
    Part part;   // written instead of out where its sums are not null: slices of a shard
};

// The larger; NaN where one of them is.
__device__ __forceinline__ float most_or_nan(float a, float b) { return a > b || a != a ? a : b; }

// A wave for each row: lists, sums and logits are read side by side, then the finish.  8192 rows of 8 shards with 20 listed tokens 12 us, 16 rows of
// slices 4 us.
template <int PLACES> __global__ __launch_bounds__(64) void distill_join_kernel(Join a)
{
    __shared__ int32_t seen[64 * PLACES];
    __shared__ double probability[64 * PLACES];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int listed = a.list.listed;
    Sums own{-__builtin_inff(), 0.0f};
    float of_target = -__builtin_inff(), again = 0.0f;
    if (lane < a.parts) {
        const float4 s = a.in.sums[(int64_t)lane * a.n + row];
        own = {s.x, s.y};
        of_target = s.z, again = s.w;
    }
    const bool repeats = __ballot(again != 0.0f) != 0;   // (a token's places are all seen by the part that holds it)
    int32_t token[PLACES];
    float teacher[PLACES], x[PLACES];
#pragma unroll
    for (int j = 0; j < PLACES; ++j) {
        const int i = lane + 64 * j;
        token[j] = -1, teacher[j] = x[j] = -__builtin_inff();
        if (i < listed) {
            const int64_t one = token_at(a.list.tokens, a.list.list_type, row * listed + i);
            if (one >= a.first && one < a.first + a.columns) token[j] = (int32_t)one;
            teacher[j] = a.list.teacher[row * listed + i];
            if (token[j] >= 0)
#pragma unroll 8
                for (int p = 0; p < a.lists; ++p) x[j] = most_or_nan(a.in.logits[((int64_t)p * a.n + row) * listed + i], x[j]);
        }
    }
    const Sums all = wave_join(own, a.c);
    const bool no_number = __ballot(of_target != of_target) != 0;
    of_target = no_number ? __builtin_nanf("") : wave_max(of_target);
    if (!a.part.sums) {
        finish_row<PLACES>(a.out, a.list, row, lane, all, token, teacher, x, of_target, repeats, seen, probability);
        return;
    }
    if (lane == 0) a.part.sums[row] = make_float4(all.m, all.s, of_target, repeats ? 1.0f : 0.0f);
#pragma unroll
    for (int j = 0; j < PLACES; ++j)
        if (lane + 64 * j < listed) a.part.logits[row * listed + lane + 64 * j] = x[j];
}

struct Grad {
    int64_t vocab, stride, out_stride, first, whole;
    int32_t slices, width;
    int32_t past;            // written past the caches
    float scale;
    List list;
    const float *stats, *grad_loss, *grad_lse, *grad_logp;
};

// Elementwise with one exponential, bound by memory: 8192 x 128256 bf16 716 us, 4.2 GB at 5.9 TB/s; a shard's 4096 x 19008 with 128 listed places 54 us,
// 5.8 TB/s; 517 x 32003 float16 15 us.  A workgroup has its columns in registers while it looks at the places, 512 vectors of two for
// each thread: with two rounds of them 8192 x 128256 796 us, with one 757 (both written in the caches).
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void distill_grad_kernel(Grad a, const typename T::raw *logits, typename T::raw *out)
{
    constexpr int VEC = T::VEC, THREADS = 64 * WAVES, ENTRIES = (GDP_MAX_LISTED + THREADS - 1) / THREADS;
    __shared__ int32_t has_target[WAVES];   // whether a wave's places hold the target
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
    const auto column_of = [&](int64_t one) -> int32_t {   // of this slice, or -1
        const int64_t local = one < 0 ? -1 : one - a.first;
        return local >= 0 && local < vocab && local >= from && local < to ? (int32_t)local : -1;
    };
    Pack<T, VEC> p[AHEAD];
    const auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            if (v < v1 && j >= 0 && j + VEC <= vocab) p[u].load(x + j);
        }
    };
    int64_t one[ENTRIES];
    float pull[ENTRIES];
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k) {
        const int e = t + k * THREADS;
        one[k] = -1;
        if (e < listed) one[k] = token_at(a.list.tokens, a.list.list_type, row * listed + e), pull[k] = stats[HEAD + e];
        if (one[k] >= a.whole) one[k] = -1;
    }
    int64_t target = a.list.targets && a.grad_logp ? token_at(a.list.targets, a.list.target_type, row) : -1;
    if (target >= a.whole) target = -1;
    load(v0);   // (on their way while the places are looked at)
    const float m = stats[0], log_s = stats[1], m_out = stats[2], log_out = stats[3];
    const bool dead = log_s < -__FLT_MAX__, none = log_out < -__FLT_MAX__;   // no logit above -inf; none that is not listed
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
    int32_t column[ENTRIES];
    float value[ENTRIES];
    bool mine = false;
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k) {
        column[k] = column_of(one[k]);
        if (column[k] < 0) continue;
        value[k] = of_loss != 0.0f ? of_loss * pull[k] : 0.0f;
        if (of_p != 0.0f) value[k] += of_p * p_of(T::up(x[column[k]]));
        if (one[k] == target) value[k] += g, mine = true;
        value[k] *= a.scale;
    }
    const bool any = __ballot(mine) != 0;
    if ((t & 63) == 0) has_target[t >> 6] = any;
    const int32_t at_target = t == 0 ? column_of(target) : -1;
    const float again = at_target >= 0 ? grad_of(T::up(x[at_target])) + a.scale * g : 0.0f;
    __syncthreads();
    for (int base = v0; base < v1; base += THREADS * AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            if (v >= v1) continue;
            if (j >= 0 && j + VEC <= vocab) {
                float f[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = grad_of(p[u][i]);
                p[u].set(f);
                if (a.past)
                    p[u].store_past(y + j);
                else
                    p[u].store(y + j);
            } else {
                for (int i = 0; i < VEC; ++i)
                    if (j + i >= 0 && j + i < vocab) y[j + i] = T::down(grad_of(T::up(x[j + i])));
            }
        }
        if (base + THREADS * AHEAD < v1) load(base + THREADS * AHEAD);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k)
        if (column[k] >= 0) y[column[k]] = T::down(value[k]);
    if (at_target >= 0) {
        bool is_listed = false;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) is_listed |= has_target[w] != 0;
        if (!is_listed) y[at_target] = T::down(again);
    }
}

// ---- host ----
// Figures that stand side by side were measured in one way, behind each other.  Some are of graphs that were replayed after a wait, which takes up to a tenth
// longer than on a busy device: they are for holding against each other.
//
// How a row is shared out: slices of 512 vectors (8 KB) at least, a workgroup for each core, and no more columns in a slice than LDS has bits
// for.  A slice is read by eight waves where there are few, else by four.  Bf16, 20 listed tokens, with 1024 workgroups of four waves and
// with 256 of eight: 333 x 32003 (float32) 16.3 and 13.9 us, 512 x 128256 33.1 and 29.9, 700 x 32000 18.5 and 16.2, 16 x 128256 9.8 and 9.7; eight
// for 2048 x 50257 56 us, four 53.
constexpr int64_t CORES = 256, MANY_GROUPS = 1024;
struct Split {
    int slices, width;
};
Split split_of(int64_t n, int64_t vocab, int type)
{
    const int vec = 16 / size_of(type);
    const int64_t vectors = ceil_div(vocab, (int64_t)vec) + 1;   // one more where a row begins within 16 bytes
    int64_t slices = 1;
    while (slices < MOST_SLICES && n * slices < CORES && vectors / (slices * 2) >= 512) slices *= 2;
    while (slices < MOST_SLICES && ceil_div(vectors, slices) * vec > MOST_BITS) slices *= 2;
    const int64_t width = ceil_div(vectors, slices);
    return {(int)ceil_div(vectors, width), (int)width};
}
// The last of the caches has 256 MB.  Logits that do not fit it are read past the caches, 8192 x 128256 bf16 363 us and 320; what does is read again by the
// gradient: 2048 x 50257 bf16 forward and backward 99 us, 109 with reads past the caches.  Gradients of half as much are written past them:
// 8192 x 128256 757 and 728 (here each result in memory of its own).
constexpr int64_t READ_PAST = 256 << 20, WRITE_PAST = 128 << 20;
// Whether rows are finished by a kernel of their own: those in slices, and, of lists with more than a place for each lane, whose finish holds
// registers that the scan could read with, those that take longer than a launch.  8192 x 128256 bf16 with 100 listed tokens 362 us, 399 where
// the scan finishes them, 4096 x 19008 with 128 57 and 63, 700 x 32000 23 and 23; but 2050 x 1000 with 100 14 and 10.
bool by_join(const Split &s, int64_t n, int64_t vocab, int listed) { return s.slices > 1 || (listed > 64 && n * vocab >= 1 << 25); }
static_assert(READ_PAST / 4 >= 1 << 25, "rows that are read past the caches are joined");
size_t sums_bytes(int64_t parts, int64_t n) { return round_up((size_t)parts * n * 16, 256); }
size_t part_bytes(int64_t parts, int64_t n, int listed) { return sums_bytes(parts, n) + round_up((size_t)n * listed * 4, 256); }
Part part_at(void *p, int64_t parts, int64_t n)
{
    return {static_cast<float4 *>(p), reinterpret_cast<float *>(static_cast<char *>(p) + sums_bytes(parts, n))};
}

// Rows of up to so many vectors (16 KB; gradients 4 KB), and at least so many of them: a wave for each row instead of four.  32089 x 1180 bf16 61 us, 99 with
// four waves, the gradient 49 and 65; 10350 x 1638 float32 31 and 35, its gradient (410 vectors) 42 and 31.
constexpr int SHORT = 1024, SHORT_GRAD = 256, SHORT_ROWS = 2048;
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
    const bool past = s.n * s.vocab * size_of(type) >= READ_PAST;
    return with_type(type, [&](auto T) {
        using TT = decltype(T);
        const auto *x = static_cast<const typename TT::raw *>(logits);
        const dim3 grid((unsigned)(s.n * split.slices));
        const size_t lds = round_up(ceil_div((size_t)split.width * TT::VEC, (size_t)32) * 4, 16);
        const auto with = [&](auto PAST, auto WAVES) {
            constexpr int waves = WAVES.value;
            if (s.list.listed <= 64) return launch(who, distill_scan_kernel<TT, 1, true, PAST.value, waves>, grid, 64 * waves, lds, stream, s, x);
            if constexpr (!PAST.value)   // (rows that are read past the caches are joined)
                if (!s.part.sums) return launch(who, distill_scan_kernel<TT, 4, true, false, waves>, grid, 64 * waves, lds, stream, s, x);
            return launch(who, distill_scan_kernel<TT, 4, false, PAST.value, waves>, grid, 64 * waves, lds, stream, s, x);
        };
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 4> four;
        const std::integral_constant<int, 8> eight;
        if (split.slices == 1 && s.n >= SHORT_ROWS && split.width <= SHORT) return with(std::false_type{}, one);
        if (s.n * split.slices < MANY_GROUPS) return past ? with(std::true_type{}, eight) : with(std::false_type{}, eight);
        return past ? with(std::true_type{}, four) : with(std::false_type{}, four);
    });
}
int join(const Join &j, const char *who, void *stream)
{
    const dim3 grid((unsigned)j.n);
    return j.list.listed <= 64 ? launch(who, distill_join_kernel<1>, grid, 64, 0, stream, j) : launch(who, distill_join_kernel<4>, grid, 64, 0, stream, j);
}
// Rows, or their slices, and what joins them.
int rows(Scan s, const void *logits, int type, void *workspace, size_t bytes, const char *who, void *stream)
{
    const Split split = split_of(s.n, s.vocab, type);
    if (s.n * split.slices > MOST_GROUPS) return gdp_fail(GDP_E_BADARG, "gdp_distill: too many rows of so many columns");
    if (split.slices == 1 && (s.part.sums || !by_join(split, s.n, s.vocab, s.list.listed))) return scan(s, logits, type, split, who, stream);
    if (!workspace || !aligned(workspace, 256) || bytes < part_bytes(split.slices, s.n, s.list.listed))
        return gdp_fail(GDP_E_BADARG, "gdp_distill: the workspace is smaller than gdp_distill_workspace says, or not aligned to 256 bytes");
    const int64_t columns = s.out.whole - s.first < s.vocab ? s.out.whole - s.first : s.vocab;
    Join j{s.n, s.first, columns, split.slices, 1, s.c, s.list, part_at(workspace, split.slices, s.n), s.out, s.part};
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
    *bytes = by_join(s, n, vocab, listed) ? part_bytes(s.slices, n, listed) : 0;
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
    if (d->whole_vocab < 0) return gdp_fail(GDP_E_BADARG, "gdp_distill: whole_vocab is negative");
    if (const int rc = check_scale(d->scale)) return rc;
    if (d->n == 0) return GDP_OK;
    const List list{d->tokens, d->targets, d->teacher, d->listed, d->list_type, d->target_type};
    if (const int rc = check_list(list)) return rc;
    if (!d->sums || !aligned(d->sums, 16) || !d->listed_logits || !aligned(d->listed_logits, 4))
        return gdp_fail(GDP_E_BADARG, "gdp_distill: null pointer, or sums not aligned to 16 bytes");
    if (const int rc = check_logits(d->logits, d->n, d->vocab, d->logits_stride, d->logits_type, false)) return rc;
    Out out{};
    out.whole = d->whole_vocab ? d->whole_vocab : INT32_MAX;
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
    return join({d->n, 0, d->vocab, d->parts, d->parts, d->scale * LOG2E, list, in, out, {}}, "gdp_distill_join", stream);
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
    // A workgroup has its columns in registers; more than once where the grid would be too large.
    const bool by_waves = d->n >= SHORT_ROWS && vectors <= SHORT_GRAD;
    int64_t width = by_waves ? SHORT_GRAD : THREADS * AHEAD;
    while (d->n * ceil_div(vectors, width) > MOST_GROUPS) width *= 2;
    const int64_t slices = ceil_div(vectors, width);
    const Grad g{d->vocab, d->logits_stride, d->out_stride, d->first, d->whole_vocab, (int32_t)slices, (int32_t)width,
                 d->n * d->vocab * size_of(d->logits_type) >= WRITE_PAST, d->scale, list, d->stats,
                 d->grad_loss, d->grad_lse, d->grad_logp};
    return with_type(d->logits_type, [&](auto T) {
        using TT = decltype(T);
        const auto *x = static_cast<const typename TT::raw *>(d->logits);
        auto *y = static_cast<typename TT::raw *>(d->out);
        const dim3 grid((unsigned)(d->n * slices));
        return by_waves ? launch("gdp_distill_backward", distill_grad_kernel<TT, 1>, grid, 64, 0, stream, g, x, y)
                        : launch("gdp_distill_backward", distill_grad_kernel<TT, THREADS / 64>, grid, THREADS, 0, stream, g, x, y);
    });
}
