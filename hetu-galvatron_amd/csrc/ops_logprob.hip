// Log probabilities of given tokens, entropy and the most likely tokens of each row of logits, and the gradient.
//
// Forward, one pass over the logits.  With c = scale * log2(e) a thread keeps of what it has read the largest logit m, s = sum of
// 2^(c (x - m)) and t = sum of 2^d * d over the exponents d = c (x - m); a new largest logit m' multiplies s by
// f = 2^(c (m - m')) and makes t f (t + c (m - m') s).  Then lse = scale * m + ln s and, since ln p = d ln 2 - ln s,
// entropy = ln s - ln 2 * t / s: two terms of one sign, nothing cancels.
//
// The most likely tokens cost the pass one write to LDS for each quad of lanes: the largest logit of each chunk of 64 bytes.  Of the
// largest logits that the 128 pairs of lanes have seen, the k-th largest is a bound: k logits reach it, so only chunks that do are
// read again, 22 for k = 20 where logits differ.  Where they do not (a row of equal logits, or with less than k that are not ruled
// out) the bound leaves too many; then the k chunks that come first by (largest logit, then number) are taken one by one: if one
// of the k largest logits lay in another chunk, k chunks would each hold a logit that comes before it.
//
// A row is one workgroup, or, where there are few rows, several workgroups of a slice each, whose results a second kernel joins; the
// same kernel joins the shards of a vocabulary.
#include "ops_common.h"

#include <type_traits>

namespace {
using namespace ops;

constexpr int THREADS = 256;
constexpr int AHEAD = 4;                 // reads of 16 bytes in flight for each thread
constexpr int MOST_CHUNKS = 8192;        // of a slice whose largest logits are asked for: 33 KB of LDS
constexpr int MOST_CHOSEN = 128;         // chunks that are read again together (by the bound), 64 where they are taken one by one
static_assert(MOST_CHOSEN >= GDP_MAX_TOP && GDP_MAX_TOP <= 64, "taken one by one; as many logits are seen apart");
constexpr int MOST_SLICES = 64;          // a lane of the joining wave for each
// Of a gradient from lse alone: below it lse is rounded by 1 or more, and exp(z - lse), which should be a share of 1, by a factor of e or
// more.  Only masks lie there (-1e9, float32's or bfloat16's lowest value): their rows get zeros.
constexpr float NO_DIGITS = -16777216.0f;

// Order of logits as whole numbers: -inf and NaN lowest, equal ones equal (-0 is 0); 0 is none of them.
__device__ __forceinline__ uint32_t key_of(float x)
{
    x = x == x ? x + 0.0f : -__builtin_inff();
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k)
{
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Sums of a part of a row.
struct Sums {
    float m, s, t;
};
// (a part without any probability has s = t = 0 and m = -inf)
__device__ __forceinline__ Sums rescaled(Sums a, float m, float c)
{
    const float d = c * (finite_or_0(a.m) - finite_or_0(m));
    const float f = exp2_fast(d);
    if (a.s == 0.0f) return {m, 0.0f, 0.0f};
    return {m, a.s * f, f == 0.0f ? 0.0f : f * fmaf(d, a.s, a.t)};
}
__device__ __forceinline__ Sums wave_join(Sums a, float c)
{
    const float m = wave_max(a.m);
    a = rescaled(a, m, c);
    return {m, wave_sum(a.s), wave_sum(a.t)};
}

struct Out {
    float *logp, *lse, *entropy, *top_logp;
    int64_t *top_tokens;
    float2 *row_stats;   // or null
};
struct Part {   // of a slice or a shard: [parts][n]
    float4 *stats;
    float *logits;
    int32_t *tokens;
};

struct Scan {
    int64_t n, vocab, stride, first, whole;
    int32_t token_type, top, slices;
    int32_t width;       // vectors of a slice, a multiple of 4
    int32_t per_super;   // chunks of a super, odd
    int32_t most_chosen; // chunks that the bound may leave
    float scale, c;
    const void *tokens;
    Out out;
    Part part;
};

__device__ __forceinline__ void finish_row(const Out &o, int64_t row, Sums a, float x, bool has_token, float scale)
{
    const float ln_s = logf(a.s), lse = a.s == 0.0f ? -__builtin_inff() : fmaf(a.m, scale, ln_s);
    o.lse[row] = lse;
    o.entropy[row] = a.s == 0.0f ? 0.0f : ln_s - LN2 * (a.t / a.s);
    if (o.row_stats) o.row_stats[row] = make_float2(a.m, ln_s);
    // (x - m) has no rounding where the token is likely, so a probability near 1 keeps its digits
    o.logp[row] = !has_token ? 0.0f : a.s == 0.0f ? -__builtin_inff() : fmaf(x - a.m, scale, -ln_s);
}
__device__ __forceinline__ float top_logp(float x, float m, float s, float scale)
{
    return s == 0.0f ? -__builtin_inff() : fmaf(x - m, scale, -logf(s));
}

// Bound by memory where rows are long: 8192 x 128256 bf16 in 364 us, 2.1 GB at 5.8 TB/s; 4096 x 50257 float32 with 5 alternatives in 158 us, 5.2
// TB/s; a shard's 8192 x 16032 bf16 53 us, 4.9 TB/s.  16 x 128256 bf16 with 20 alternatives: 10 us in 256 workgroups, 5 of them without alternatives: barriers and waits.
// Of short rows the choice takes longer than the reading: 15744 x 2304 bf16 23 us, 70 with 20 alternatives.
// WAVES: four to a row or slice; one where rows are short and many.
template <typename T, bool TOP, int WAVES> __global__ __launch_bounds__(64 * WAVES) void logprob_scan_kernel(Scan a, const typename T::raw *__restrict__ logits)
{
    constexpr int VEC = T::VEC, THREADS = 64 * WAVES;
    constexpr int SEEN = WAVES == 1 ? 64 : THREADS / 2;   // lanes, or pairs of lanes, whose largest logits give the bound
    extern __shared__ __align__(16) float chunk_max[];   // [64 * per_super], then their keys
    __shared__ Sums of_wave[WAVES];
    __shared__ int32_t chosen[MOST_CHOSEN], n_chosen, n_found;
    __shared__ __align__(16) uint32_t seen[SEEN];
    __shared__ uint32_t least;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t row = blockIdx.x / a.slices;
    const int slice = (int)(blockIdx.x % a.slices);
    const typename T::raw *const x = logits + row * a.stride;
    // Vectors are counted from the 16 bytes that the row begins in: the first and the last may be cut.
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(typename T::raw));
    const int vocab = (int)a.vocab, vectors = (vocab + off + VEC - 1) / VEC;
    const int v0 = slice * a.width, v1 = v0 + a.width < vectors ? v0 + a.width : vectors;
    const float c = a.c;
    Sums own{-__builtin_inff(), 0.0f, 0.0f};
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
            float b = p[u][0];
#pragma unroll
            for (int i = 1; i < VEC; ++i) b = fmaxf(b, p[u][i]);
            most = fmaxf(most, b);
            if constexpr (TOP) {
                b = fmaxf(b, dpp<QUAD_SWAP1>(b, b));
                b = fmaxf(b, dpp<QUAD_SWAP2>(b, b));
                const int v = base + u * THREADS + t;
                if ((t & 3) == 0 && v < v1) chunk_max[(v - v0) >> 2] = b;
            }
        }
        own = rescaled(own, most, c);
        const float from = finite_or_0(most);   // (subtracted first: a row may hold a type's lowest value alone)
        float sum = 0.0f, sum_t = 0.0f;         // of these reads: a row's sums then are of few terms each
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = (p[u][i] - from) * c, e = exp2_fast(d);
                sum += e;
                sum_t = fmaf(e, fmaxf(d, -1e4f), sum_t);   // 2^-inf * -inf would be NaN; below -1e4 the product is 0
            }
        }
        own.s += sum, own.t += sum_t;
    }
    if constexpr (TOP) {
        if constexpr (WAVES == 1) {
            seen[t] = key_of(own.m);
        } else {
            const float b = fmaxf(own.m, dpp<QUAD_SWAP1>(own.m, own.m));
            if ((t & 1) == 0) seen[t >> 1] = key_of(b);
        }
        if (t == 0) n_chosen = n_found = 0;
    }
    own = wave_join(own, c);
    if (lane == 0) of_wave[wave] = own;
    __syncthreads();
    float m = of_wave[0].m;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, of_wave[w].m);
    Sums all{m, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const Sums r = rescaled(of_wave[w], m, c);
        all.s += r.s, all.t += r.t;
    }
    const int64_t at = (int64_t)slice * a.n + row;   // of the row's part
    if (t == 0) {
        const int64_t token = token_at(a.tokens, a.token_type, row);
        const int64_t local = token - a.first;
        const bool here = token >= 0 && token < a.whole && local >= (int64_t)v0 * VEC - off && local < (int64_t)v1 * VEC - off && local >= 0 && local < vocab;
        const float of_token = here ? T::up(x[local]) : -__builtin_inff();
        if (a.part.stats)
            a.part.stats[at] = make_float4(all.m, all.s, all.t, of_token);
        else
            finish_row(a.out, row, all, of_token, here, a.scale);
    }
    if constexpr (TOP) {
        const int chunks = v1 > v0 ? (v1 - v0 + 3) / 4 : 0, per = a.per_super;
        // The bound, in each wave: the least of the largest logits seen that fewer than `top` exceed.  (What follows runs once: it is
        // kept in loops of few instructions, which are fetched sooner than unrolled ones.)
        uint32_t bound;
        {
            const uint4 *const all_seen = reinterpret_cast<const uint4 *>(seen);
            bound = ~0u;
#pragma unroll
            for (int mine = lane; mine < SEEN; mine += 64) {
                const uint32_t one = seen[mine];
                int larger = 0;
#pragma unroll 4
                for (int i = 0; i < SEEN / 4; ++i) {
                    const uint4 q = all_seen[i];
                    larger += (q.x > one) + (q.y > one) + (q.z > one) + (q.w > one);
                }
                bound = min(bound, larger < a.top ? one : ~0u);
            }
            bound = wave_min(bound);
        }
#pragma unroll 1
        for (int i = t; i < chunks; i += THREADS)
            if (key_of(chunk_max[i]) >= bound) {
                const int at_list = atomicAdd(&n_chosen, 1);
                if (at_list < a.most_chosen) chosen[at_list] = i;
            }
        __syncthreads();
        if (n_chosen > a.most_chosen) {
            uint32_t *const key = reinterpret_cast<uint32_t *>(chunk_max);
            for (int i = t; i < 64 * per; i += THREADS) key[i] = i < chunks ? key_of(chunk_max[i]) : 0u;
            __syncthreads();
            if (wave == 0) {
                // A lane has `per` neighbouring chunks, a super; their number is odd, so that lanes read from different banks.
                uint32_t best = 0;
                for (int i = 0; i < per; ++i) best = max(best, key[lane * per + i]);
                int count = 0;
                uint32_t last = 0;
                for (; count < a.top; ++count) {
                    const uint32_t most = wave_max(best);
                    if (most == 0) break;
                    last = most;
                    const int super = __builtin_ctzll(__ballot(best == most));
                    uint32_t rest = 0;
                    bool taken = false;
                    for (int i = 0; i < per; i += 64) {
                        const int at_key = super * per + i + lane;
                        uint32_t k = i + lane < per ? key[at_key] : 0u;
                        if (!taken) {
                            const uint64_t equal = __ballot(k == most);
                            if (equal) {
                                taken = true;
                                const int w = __builtin_ctzll(equal);
                                if (lane == w) {
                                    k = 0;
                                    key[at_key] = 0;
                                    chosen[count] = super * per + i + w;
                                }
                            }
                        }
                        rest = max(rest, k);
                    }
                    rest = wave_max(rest);
                    if (lane == super) best = rest;
                }
                if (lane == 0) {
                    n_chosen = count;
                    least = count == a.top ? last : 0u;   // top chunks have a logit of this or more each
                }
            }
            __syncthreads();
            bound = least;
        }
        // Their logits that can be among the first, in any order; the largest logits of the chunks are not needed any more.
        uint64_t *const found = reinterpret_cast<uint64_t *>(chunk_max);
#pragma unroll 1
        for (int i = t; i < n_chosen * 4; i += THREADS) {
            const int v = v0 + 4 * chosen[i >> 2] + (i & 3), j = v * VEC - off;
            uint32_t k[VEC];
            int count = 0;
            if (j >= 0 && j + VEC <= vocab) {
                Pack<T, VEC> p;
                p.load(x + j);
#pragma unroll
                for (int e = 0; e < VEC; ++e) k[e] = key_of(p[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) k[e] = j + e >= 0 && j + e < vocab ? key_of(T::up(x[j + e])) : 0u;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) count += k[e] != 0 && k[e] >= bound;   // (the bound is 0 where there are fewer than `top`)
            if (count) {
                int to = atomicAdd(&n_found, count);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (k[e] != 0 && k[e] >= bound) found[to++] = (uint64_t)k[e] << 32 | (uint32_t)~(j + e);
            }
        }
        __syncthreads();
        const int n = n_found;
        for (int i = t; i < n; i += THREADS) {
            const uint64_t one = found[i];
            int place = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) place += found[j] > one;
            if (place < a.top) {
                const float logit = of_key((uint32_t)(one >> 32));
                const int64_t token = a.first + (int32_t)~(uint32_t)one;
                if (a.part.stats) {
                    a.part.logits[at * a.top + place] = logit;
                    a.part.tokens[at * a.top + place] = (int32_t)token;
                } else {
                    a.out.top_logp[row * a.top + place] = top_logp(logit, all.m, all.s, a.scale);
                    a.out.top_tokens[row * a.top + place] = token;
                }
            }
        }
        if (a.part.stats)
            for (int i = n + t; i < a.top; i += THREADS) {
                a.part.logits[at * a.top + i] = -__builtin_inff();
                a.part.tokens[at * a.top + i] = -1;
            }
    }
}

struct Join {
    int64_t n, whole;
    int32_t parts, top, first, token_type;   // `first` of each list for the bound
    int32_t reach;       // logits that LDS has room for behind the lists
    float scale, c;
    const void *tokens;
    Part in;
    Out out;
    Part part;   // written instead of out where its stats are not null: slices of a shard
};

// A workgroup joins a row: a lane of each wave for each part.  Of the lists of the most likely tokens, which are sorted, the first
// few of each, twice as many as are asked for in all, give a bound that `top` of them reach: what does not reach it is left out, and
// what does finds its place by looking at all that do.
// A launch and four waits for memory or barriers: 16 rows of 16 parts and 20 alternatives 7 us, 3 without alternatives.
static_assert(GDP_MAX_TOP <= 64 && MOST_SLICES <= 64, "a lane for each");
constexpr int JOIN_THREADS = 256;
__global__ __launch_bounds__(JOIN_THREADS) void logprob_join_kernel(Join a)
{
    extern __shared__ __align__(16) uint64_t lists[];   // [parts][top], then the first of each, and later those that reach the bound
    __shared__ unsigned long long bound;
    __shared__ int32_t n_found, used[GDP_MAX_TOP];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, waves = blockDim.x >> 6;
    const int64_t row = blockIdx.x;
    Sums own{-__builtin_inff(), 0.0f, 0.0f};
    float x = -__builtin_inff();
    if (lane < a.parts) {
        const float4 s = a.in.stats[(int64_t)lane * a.n + row];
        own = {s.x, s.y, s.z};
        x = s.w;
    }
    uint64_t *const found = lists + a.parts * a.top;
    const int first = a.first, some = first * a.parts;
    if (lane < a.top)   // (GDP_MAX_TOP lanes: one for each place of a list)
#pragma unroll 4
        for (int p = wave; p < a.parts; p += waves) {
            const int64_t from = ((int64_t)p * a.n + row) * a.top + lane;
            const int32_t token = a.in.tokens[from];
            const uint64_t one = token < 0 ? 0 : (uint64_t)key_of(a.in.logits[from]) << 32 | (uint32_t)~token;
            lists[p * a.top + lane] = one;
            if (lane < first) found[p * first + lane] = one;
        }
    if (t == 0) n_found = 0, bound = ~0ull;
    if (t < GDP_MAX_TOP) used[t] = 0;
    const Sums all = wave_join(own, a.c);
    x = wave_max(x);
    if (t == 0) {
        if (a.part.stats)
            a.part.stats[row] = make_float4(all.m, all.s, all.t, x);
        else {
            const int64_t token = token_at(a.tokens, a.token_type, row);
            finish_row(a.out, row, all, x, token >= 0 && token < a.whole, a.scale);
        }
    }
    if (a.top == 0) return;
    __syncthreads();
    for (int i = t; i < some; i += JOIN_THREADS) {   // the least that fewer than `top` exceed
        const uint64_t one = found[i];
        int larger = 0;
#pragma unroll 8
        for (int j = 0; j < some; ++j) larger += found[j] > one;
        if (larger < a.top) atomicMin(&bound, (unsigned long long)one);
    }
    __syncthreads();
    const uint64_t least = bound;
    if (lane < a.top)
        for (int p = wave; p < a.parts; p += waves) {
            const uint64_t one = lists[p * a.top + lane];
            if (one != 0 && one >= least) {
                const int to = atomicAdd(&n_found, 1);
                if (to < a.reach) found[to] = one;
            }
        }
    __syncthreads();
    // As parts leave them, their lists are in order and there is room for all that reach the bound.  Of a caller's lists that are not, more
    // may reach it: then all of the lists are looked at.  A token that is there twice has two places, one behind the other.
    const bool fits = n_found <= a.reach;
    const uint64_t *const from = fits ? found : lists;
    const int n = fits ? n_found : a.parts * a.top;
    const float log_s = all.s == 0.0f ? 0.0f : logf(all.s);
    const auto put = [&](int place, float logit, int32_t token) {
        if (a.part.stats) {
            a.part.logits[row * a.top + place] = logit;
            a.part.tokens[row * a.top + place] = token;
        } else {
            a.out.top_logp[row * a.top + place] = all.s == 0.0f ? -__builtin_inff() : fmaf(logit - all.m, a.scale, -log_s);
            a.out.top_tokens[row * a.top + place] = token;
        }
    };
    for (int i = t; i < n; i += JOIN_THREADS) {
        const uint64_t one = from[i];
        int place = one == 0 ? a.top : 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) place += from[j] > one;
        if (place < a.top) place += atomicAdd(&used[place], 1);
        if (place < a.top) put(place, of_key((uint32_t)(one >> 32)), (int32_t)~(uint32_t)one);
    }
    for (int i = n + t; i < a.top; i += JOIN_THREADS) put(i, -__builtin_inff(), -1);   // parts of fewer tokens than are asked for
}

struct Grad {
    int64_t vocab, stride, out_stride, first, whole;
    int32_t token_type, top, slices, width;
    float scale;
    const void *tokens;
    const float *lse, *grad_logp, *grad_lse, *entropy, *grad_entropy, *grad_top;
    const int64_t *top_tokens;
    const float *row_stats;   // [n][2], or null: by lse
};

// ln p_j = scale (x_j - m) - ln s, by the same steps as in the forward pass: a row's level cancels.  From lse alone scale x_j - lse, whose two
// terms are off by what lse is rounded by.
// out_j = scale * (delta_j - p_j (g + h (ln p_j + entropy))): elementwise, bound by memory, but for the few columns with a delta, which
// a workgroup reads first and writes again at the end (out may be the logits).  8192 x 128256 bf16 in 810 us, 4.2 GB at 5.2 TB/s.
// STATS: from row_stats; a subtraction more for each logit, 517 x 32003 f16 with entropies 16.4 us and 15.8 from lse.
template <typename T, bool ENTROPY, bool STATS>
__global__ __launch_bounds__(THREADS) void logprob_grad_kernel(Grad a, const typename T::raw *logits, typename T::raw *out)
{
    constexpr int VEC = T::VEC;
    __shared__ int64_t column[GDP_MAX_TOP + 1];
    __shared__ float delta[GDP_MAX_TOP + 1];
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x / a.slices;
    const int slice = (int)(blockIdx.x % a.slices);
    const typename T::raw *const x = logits + row * a.stride;
    typename T::raw *const y = out + row * a.out_stride;
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(typename T::raw));
    const int vocab = (int)a.vocab, vectors = (vocab + off + VEC - 1) / VEC;
    const int v0 = slice * a.width, v1 = v0 + a.width < vectors ? v0 + a.width : vectors;
    const float largest = STATS ? a.row_stats[2 * row] : 0.0f, log_sum = STATS ? a.row_stats[2 * row + 1] : a.lse[row];
    const bool dead = log_sum < (STATS ? -__FLT_MAX__ : NO_DIGITS);
    const float minus = dead ? 0.0f : -a.scale;
    const int64_t token = token_at(a.tokens, a.token_type, row);
    const float of_token = a.grad_logp && token >= 0 && token < a.whole ? a.grad_logp[row] : 0.0f;
    const int entries = 1 + a.top;
    if (t < entries) {
        column[t] = t == 0 ? (of_token != 0.0f ? token - a.first : -1) : a.top_tokens[row * a.top + t - 1] - a.first;
        delta[t] = t == 0 ? of_token : a.grad_top[row * a.top + t - 1];
    }
    __syncthreads();
    float g = of_token - (a.grad_lse ? a.grad_lse[row] : 0.0f), h = 0.0f, rest = 0.0f;
    for (int i = 1; i < entries; ++i) g += delta[i];
    if constexpr (ENTROPY) {
        h = a.grad_entropy[row];
        rest = a.entropy[row];
    }
    if (dead) g = h = rest = 0.0f;   // (all p are 0, and nothing is multiplied by them)
    const float from = dead ? 0.0f : largest, away = dead ? __builtin_inff() : log_sum;
    const auto grad_of = [&](float f) {
        const float q = fmaf(STATS ? f - from : f, a.scale, -away);
        const float p = exp2_fast(q * LOG2E);
        const float w = ENTROPY ? fmaf(h, fmaxf(q, -1e4f) + rest, g) : g;   // (p is 0 below)
        return minus * (p * w);
    };
    // the columns with a delta: theirs without it, from the logit, before anything is written
    float again = 0.0f;
    bool mine = false;
    if (t < entries) {
        const int64_t j = column[t];
        mine = j >= 0 && j < vocab && j >= (int64_t)v0 * VEC - off && j < (int64_t)v1 * VEC - off;
        if (mine) {
            float d = 0.0f;
            for (int i = 0; i < entries; ++i) d += column[i] == j ? delta[i] : 0.0f;
            again = dead ? 0.0f : grad_of(T::up(x[j])) + a.scale * d;
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
    if (mine) y[column[t]] = T::down(again);
}

// ---- host ----
// How a row is shared out: slices of 512 vectors (8 KB) at least, 1024 workgroups, and no more chunks in a slice than LDS is laid out
// for.  512 where alternatives are asked for: each slice then has some 5 us of work of its own.  128256 columns of bf16, top 0
// / 20, with 512 and 1024 workgroups: 64 rows 7.8 / 16.8 and 7.6 / 20.1 us, 300 rows 22.0 / 35.1 and 19.2 / 32.1, 512 rows
// 27.7 / 38.2 and 26.8 / 40.6.
struct Split {
    int slices, width, per_super;
};
Split split_of(int64_t n, int64_t vocab, int type, int top)
{
    const int vec = 16 / size_of(type);
    const int64_t vectors = ceil_div(vocab, (int64_t)vec) + 1;   // one more where a row begins within 16 bytes
    int64_t slices = 1;
    while (slices < MOST_SLICES && n * slices < (top ? 512 : 1024) && vectors / (slices * 2) >= 512) slices *= 2;
    if (top)
        while (slices < MOST_SLICES && ceil_div(vectors, slices) > 4 * MOST_CHUNKS) slices *= 2;
    const int64_t width = round_up((size_t)ceil_div(vectors, slices), 4);
    slices = ceil_div(vectors, width);
    const int64_t per = ceil_div(ceil_div(width, (int64_t)4), (int64_t)64) | 1;
    return {(int)slices, (int)width, (int)per};
}
size_t part_bytes(int64_t parts, int64_t n, int top) { return round_up((size_t)parts * n * 16, 256) + 2 * round_up((size_t)parts * n * top * 4, 256); }
Part part_at(void *p, int64_t parts, int64_t n, int top)
{
    char *const w = static_cast<char *>(p);
    const size_t a = round_up((size_t)parts * n * 16, 256), b = round_up((size_t)parts * n * top * 4, 256);
    return {reinterpret_cast<float4 *>(w), reinterpret_cast<float *>(w + a), reinterpret_cast<int32_t *>(w + a + b)};
}

// Rows of up to so many vectors (32 KB), and at least so many of them: a wave for each row instead of four.  32768 rows of 1000 bf16 25 us,
// 89 with four waves; of 8192 bf16, top 5, 181 and 214; but 8192 of 16384, top 5, 89 and 85.
constexpr int SHORT = 2048, SHORT_ROWS = 2048;
constexpr int64_t MOST_ROWS = (int64_t)1 << 21, MOST_GROUPS = (int64_t)1 << 23;   // a grid has less than 2^32 threads
int check(int64_t n, int64_t vocab, int64_t first, int type, int token_type, int top)
{
    if (n < 0 || vocab < 1 || first < 0) return gdp_fail(GDP_E_BADARG, "gdp_logprob: a size is negative, or there are no columns");
    if (n > MOST_ROWS || vocab > GDP_MAX_VOCAB || first > INT32_MAX - vocab)
        return gdp_fail(GDP_E_BADARG, "gdp_logprob: more than 2^21 rows or GDP_MAX_VOCAB columns, or a token above 2^31");
    if (!type_ok(type) || !token_type_ok(token_type)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: unknown element type");
    if (top < 0 || top > GDP_MAX_TOP) return gdp_fail(GDP_E_BADARG, "gdp_logprob: top must be 0 to GDP_MAX_TOP");
    if (n * split_of(n, vocab, type, top).slices > MOST_GROUPS) return gdp_fail(GDP_E_BADARG, "gdp_logprob: too many rows for alternatives of so many columns");
    return GDP_OK;
}
int check_scale(float scale)
{
    return scale > 0.0f && scale < 1e30f ? GDP_OK : gdp_fail(GDP_E_BADARG, "gdp_logprob: scale must be positive and below 1e30");
}
int check_logits(const void *p, int64_t n, int64_t vocab, int64_t stride, int type, const void *tokens, int token_type, bool written)
{
    if (!p || !tokens) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null pointer");
    if (!rows_ok(n, vocab, stride, written)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: a row stride is negative, too large, or below the width of rows that are written");
    if (!aligned(p, size_of(type)) || !aligned(tokens, token_type == GDP_I64 ? 8 : 4))
        return gdp_fail(GDP_E_BADARG, "gdp_logprob: a pointer is not aligned to its elements");
    return GDP_OK;
}

int scan(Scan s, const void *logits, int type, const Split &split, const char *who, void *stream)
{
    s.slices = split.slices, s.width = split.width, s.per_super = split.per_super;
    s.c = s.scale * LOG2E;
    size_t lds = (size_t)64 * split.per_super * 4;
    s.most_chosen = s.top <= 24 ? MOST_CHOSEN / 2 : MOST_CHOSEN;   // (for 24 the bound leaves 27 chunks, for 64 it leaves 89; LDS for 64 lets 8 workgroups on a core)
    const size_t found = (size_t)s.most_chosen * 4 * (16 / size_of(type)) * 8;
    if (lds < found) lds = found;   // (a row of fewer chunks finds no more than they have)
    const size_t whole = round_up((size_t)split.width * 16 / size_of(type) * 8, 16);
    if (lds > whole && whole >= (size_t)64 * split.per_super * 4) lds = whole;
    return with_type(type, [&](auto T) {
        using TT = decltype(T);
        const auto *x = static_cast<const typename TT::raw *>(logits);
        const dim3 grid((unsigned)(s.n * split.slices));
        if (split.slices == 1 && s.n >= SHORT_ROWS && split.width <= SHORT)
            return s.top ? launch(who, logprob_scan_kernel<TT, true, 1>, grid, 64, lds, stream, s, x)
                         : launch(who, logprob_scan_kernel<TT, false, 1>, grid, 64, 0, stream, s, x);
        return s.top ? launch(who, logprob_scan_kernel<TT, true, 4>, grid, THREADS, lds, stream, s, x)
                     : launch(who, logprob_scan_kernel<TT, false, 4>, grid, THREADS, 0, stream, s, x);
    });
}
int join(Join j, const char *who, void *stream)
{
    j.first = (2 * j.top + j.parts - 1) / j.parts;
    if (j.first > j.top) j.first = j.top;
    // At most `top` of the lists' first logits reach the bound, so at most top / first lists, half of them, reach it with all of those and
    // can go on to the end; the others end among them.
    j.reach = j.parts * j.top / 2 + 2 * j.top + j.parts;
    return launch(who, logprob_join_kernel, dim3((unsigned)j.n), j.top ? JOIN_THREADS : 64, ((size_t)j.parts * j.top + j.reach) * 8, stream, j);
}

}  // namespace

extern "C" int gdp_logprob_workspace(int64_t n, int64_t vocab, int32_t logits_type, int32_t top, size_t *bytes)
{
    gdp_clear_error();
    if (!bytes) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
    if (const int rc = check(n, vocab, 0, logits_type, GDP_I64, top)) return rc;
    const Split s = split_of(n, vocab, logits_type, top);
    *bytes = s.slices > 1 ? part_bytes(s.slices, n, top) : 0;
    return GDP_OK;
}

static int forward_rows(const gdp_logprob *l, float *row_stats, void *stream)
{
    if (!aligned(row_stats, 8)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: row_stats must be aligned to 8 bytes");
    if (const int rc = check(l->n, l->vocab, 0, l->logits_type, l->token_type, l->top)) return rc;
    if (l->top > l->vocab) return gdp_fail(GDP_E_BADARG, "gdp_logprob: top is above the number of columns");
    if (const int rc = check_scale(l->scale)) return rc;
    if (l->n == 0) return GDP_OK;
    if (const int rc = check_logits(l->logits, l->n, l->vocab, l->logits_stride, l->logits_type, l->tokens, l->token_type, false)) return rc;
    if (!l->logp || !l->lse || !l->entropy || (l->top && (!l->top_logp || !l->top_tokens))) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null pointer");
    const Split split = split_of(l->n, l->vocab, l->logits_type, l->top);
    const Out out{l->logp, l->lse, l->entropy, l->top_logp, l->top_tokens, reinterpret_cast<float2 *>(row_stats)};
    Scan s{l->n, l->vocab, l->logits_stride, 0, l->vocab, l->token_type, l->top, 1, 0, 1, 0, l->scale, 0.0f, l->tokens, out, {}};
    if (split.slices == 1) return scan(s, l->logits, l->logits_type, split, "gdp_logprob_forward", stream);
    if (!aligned(l->workspace, 256) || !l->workspace || l->workspace_bytes < part_bytes(split.slices, l->n, l->top))
        return gdp_fail(GDP_E_BADARG, "gdp_logprob: the workspace is smaller than gdp_logprob_workspace says, or not aligned to 256 bytes");
    s.part = part_at(l->workspace, split.slices, l->n, l->top);
    if (const int rc = scan(s, l->logits, l->logits_type, split, "gdp_logprob_forward", stream)) return rc;
    return join({l->n, l->vocab, split.slices, l->top, 0, l->token_type, 0, l->scale, l->scale * LOG2E, l->tokens, s.part, out, {}}, "gdp_logprob_forward", stream);
}

extern "C" int gdp_logprob_forward(const gdp_logprob *l, void *stream)
{
    gdp_clear_error();
    return l ? forward_rows(l, nullptr, stream) : gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
}

extern "C" int gdp_logprob_forward_stats(const gdp_logprob_stats *l, void *stream)
{
    gdp_clear_error();
    if (!l || (!l->row_stats && l->given.n != 0)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
    return forward_rows(&l->given, l->row_stats, stream);
}

extern "C" int gdp_logprob_parts(const gdp_logprob_part *l, void *stream)
{
    gdp_clear_error();
    if (!l) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
    if (const int rc = check(l->n, l->vocab, l->first, l->logits_type, l->token_type, l->top)) return rc;
    if (const int rc = check_scale(l->scale)) return rc;
    if (l->n == 0) return GDP_OK;
    if (const int rc = check_logits(l->logits, l->n, l->vocab, l->logits_stride, l->logits_type, l->tokens, l->token_type, false)) return rc;
    if (!l->stats || !aligned(l->stats, 16) || (l->top && (!l->top_logits || !l->top_tokens)))
        return gdp_fail(GDP_E_BADARG, "gdp_logprob: null pointer, or stats not aligned to 16 bytes");
    const Split split = split_of(l->n, l->vocab, l->logits_type, l->top);
    const Part own{reinterpret_cast<float4 *>(l->stats), l->top_logits, l->top_tokens};
    Scan s{l->n, l->vocab, l->logits_stride, l->first, (int64_t)INT32_MAX, l->token_type, l->top, 1, 0, 1, 0, l->scale, 0.0f, l->tokens, {}, own};
    if (split.slices == 1) return scan(s, l->logits, l->logits_type, split, "gdp_logprob_parts", stream);
    if (!aligned(l->workspace, 256) || !l->workspace || l->workspace_bytes < part_bytes(split.slices, l->n, l->top))
        return gdp_fail(GDP_E_BADARG, "gdp_logprob: the workspace is smaller than gdp_logprob_workspace says, or not aligned to 256 bytes");
    s.part = part_at(l->workspace, split.slices, l->n, l->top);
    if (const int rc = scan(s, l->logits, l->logits_type, split, "gdp_logprob_parts", stream)) return rc;
    return join({l->n, (int64_t)INT32_MAX, split.slices, l->top, 0, l->token_type, 0, l->scale, l->scale * LOG2E, l->tokens, s.part, {}, own}, "gdp_logprob_parts", stream);
}

static int join_rows(const gdp_logprob_joint *l, float *row_stats, void *stream)
{
    if (!aligned(row_stats, 8)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: row_stats must be aligned to 8 bytes");
    if (l->n < 0 || l->n > MOST_ROWS || l->vocab < 1 || l->vocab > INT32_MAX) return gdp_fail(GDP_E_BADARG, "gdp_logprob: a size is out of range");
    if (l->parts < 1 || l->parts > GDP_MAX_LOGPROB_PARTS) return gdp_fail(GDP_E_BADARG, "gdp_logprob: parts must be 1 to GDP_MAX_LOGPROB_PARTS");
    if (l->top < 0 || l->top > GDP_MAX_TOP || l->top > l->vocab) return gdp_fail(GDP_E_BADARG, "gdp_logprob: top must be 0 to GDP_MAX_TOP and at most the vocabulary");
    if (!token_type_ok(l->token_type)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: unknown element type");
    if (const int rc = check_scale(l->scale)) return rc;
    if (l->n == 0) return GDP_OK;
    if (!l->tokens || !l->stats || !l->logp || !l->lse || !l->entropy || (l->top && (!l->top_logits || !l->top_tokens || !l->top_logp || !l->out_tokens)))
        return gdp_fail(GDP_E_BADARG, "gdp_logprob: null pointer");
    if (!aligned(l->stats, 16) || !aligned(l->tokens, l->token_type == GDP_I64 ? 8 : 4))
        return gdp_fail(GDP_E_BADARG, "gdp_logprob: stats not aligned to 16 bytes, or tokens not to their elements");
    const Part in{reinterpret_cast<float4 *>(const_cast<float *>(l->stats)), const_cast<float *>(l->top_logits), const_cast<int32_t *>(l->top_tokens)};
    return join({l->n, l->vocab, l->parts, l->top, 0, l->token_type, 0, l->scale, l->scale * LOG2E, l->tokens, in, {l->logp, l->lse, l->entropy, l->top_logp, l->out_tokens, reinterpret_cast<float2 *>(row_stats)}, {}},
                "gdp_logprob_join", stream);
}

extern "C" int gdp_logprob_join(const gdp_logprob_joint *l, void *stream)
{
    gdp_clear_error();
    return l ? join_rows(l, nullptr, stream) : gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
}

extern "C" int gdp_logprob_join_stats(const gdp_logprob_joint_stats *l, void *stream)
{
    gdp_clear_error();
    if (!l || (!l->row_stats && l->given.n != 0)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
    return join_rows(&l->given, l->row_stats, stream);
}

static int backward_rows(const gdp_logprob_grad *l, const float *row_stats, void *stream)
{
    if (!aligned(row_stats, 8)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: row_stats must be aligned to 8 bytes");
    if (const int rc = check(l->n, l->vocab, l->first, l->logits_type, l->token_type, l->top)) return rc;
    if (l->whole_vocab < 1) return gdp_fail(GDP_E_BADARG, "gdp_logprob: a size is out of range");
    if (const int rc = check_scale(l->scale)) return rc;
    if (l->n == 0) return GDP_OK;
    if (const int rc = check_logits(l->logits, l->n, l->vocab, l->logits_stride, l->logits_type, l->tokens, l->token_type, false)) return rc;
    if (const int rc = check_logits(l->out, l->n, l->vocab, l->out_stride, l->logits_type, l->tokens, l->token_type, true)) return rc;
    if ((!l->lse && !row_stats) || !l->entropy != !l->grad_entropy || (l->top && (!l->top_tokens || !l->grad_top))) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null pointer");
    if (l->out == l->logits && l->n > 1 && l->out_stride != l->logits_stride) return gdp_fail(GDP_E_BADARG, "gdp_logprob: a gradient in the place of the logits needs their stride");
    const int vec = 16 / size_of(l->logits_type);
    const int64_t vectors = ceil_div(l->vocab, (int64_t)vec) + 1;
    int64_t slices = 1;   // two rounds of reads for each workgroup, more where the grid would be too large
    while (vectors / slices > 2 * THREADS * AHEAD && l->n * slices < (1 << 22)) slices *= 2;
    const int64_t width = ceil_div(vectors, slices);
    slices = ceil_div(vectors, width);
    const Grad g{l->vocab, l->logits_stride, l->out_stride, l->first, l->whole_vocab, l->token_type, l->top, (int32_t)slices, (int32_t)width, l->scale,
                 l->tokens, l->lse, l->grad_logp, l->grad_lse, l->entropy, l->grad_entropy, l->grad_top, l->top_tokens, row_stats};
    return with_type(l->logits_type, [&](auto T) {
        using TT = decltype(T);
        const auto *x = static_cast<const typename TT::raw *>(l->logits);
        auto *y = static_cast<typename TT::raw *>(l->out);
        const dim3 grid((unsigned)(l->n * slices));
        const auto run = [&](auto ENTROPY, auto STATS) {
            return launch("gdp_logprob_backward", logprob_grad_kernel<TT, ENTROPY.value, STATS.value>, grid, THREADS, 0, stream, g, x, y);
        };
        const auto with = [&](auto ENTROPY) { return row_stats ? run(ENTROPY, std::true_type{}) : run(ENTROPY, std::false_type{}); };
        return l->entropy ? with(std::true_type{}) : with(std::false_type{});
    });
}

extern "C" int gdp_logprob_backward(const gdp_logprob_grad *l, void *stream)
{
    gdp_clear_error();
    return l ? backward_rows(l, nullptr, stream) : gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
}

extern "C" int gdp_logprob_backward_stats(const gdp_logprob_grad_stats *l, void *stream)
{
    gdp_clear_error();
    if (!l || (!l->row_stats && l->given.n != 0)) return gdp_fail(GDP_E_BADARG, "gdp_logprob: null argument");
    return backward_rows(&l->given, l->row_stats, stream);
}
