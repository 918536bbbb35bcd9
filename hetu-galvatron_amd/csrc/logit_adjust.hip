// Penalties for repeated tokens, biases of single tokens, a grammar's mask and a temperature on rows of logits, and the gradient.
//
// A workgroup has a slice of a row's columns.  It reads the row's history and counts the slice's tokens in a table in LDS, 4 bytes for each
// column: bit 31 for a token of the prompt, bit 30 for a token with a bias, and below them how often the token is in what was drawn.
// Then it passes over its columns once, 16 bytes at a time, with their bits of the mask and their places of the table.  Counts are whole
// numbers, so the order in which atomics add them up does not show.  Biases are kept as a list in the order they are given: a column whose bit 30
// is set adds up its own.
//
// Columns that the mask rules out are not read; where the result takes the logits' place and nothing else changes, neither read nor written.
// Bound by memory; with long histories by reading them once for each slice.
#include "ops_common.h"

#include <type_traits>

namespace {
using namespace ops;

constexpr int COLUMNS = 8192;               // of a slice; with a table 32 KB of LDS, four workgroups on a core
constexpr int threads_of(bool table) { return table ? 512 : 256; }
constexpr int HISTORY_AHEAD = 4;            // tokens of the history that a thread has in flight
constexpr uint32_t OF_PROMPT = 1u << 31, HAS_BIAS = 1u << 30, COUNT = HAS_BIAS - 1;
constexpr int64_t MOST_PLACES = COUNT;      // of a history

struct Bias {
    int32_t column;      // of the slice
    float value;
};
struct Adjust {
    int64_t vocab, stride, out_stride, grad_stride, first;
    int32_t slices;
    gdp_adjust_history history;
    const void *bias_tokens;
    const float *bias;
    int64_t bias_stride;
    int32_t biases, bias_token_type;
    const uint32_t *allowed;
    int64_t allowed_stride;
    const float *scales;
    float scale;
    int32_t in_place;        // what does not change need not be written
};

__device__ __forceinline__ int64_t at_most(const void *p, int type, int64_t row, int64_t otherwise, int64_t most)
{
    const int64_t n = p ? token_at(p, type, row) : otherwise;
    return n < 0 ? 0 : n > most ? most : n;
}

// Tokens from `begin` on, every THREADS-th, less `base`; above every column behind `end`.
template <int THREADS, int N> __device__ __forceinline__ void load_tokens(uint64_t (&to)[N], const void *tokens, int type, int64_t begin, int64_t i, int64_t end)
{
    if (type == GDP_I64) {
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (i + u * THREADS < end) to[u] = (uint64_t) static_cast<const int64_t *>(tokens)[begin + i + u * THREADS];
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (i + u * THREADS < end) to[u] = (uint64_t)(int64_t) static_cast<const int32_t *>(tokens)[begin + i + u * THREADS];
    }
}

// T: of the logits; O: of what is written, or of the gradient that is read (BACK).  TABLE: there is a history or are biases.
// A thread has all of its columns, VECTORS times 16 bytes of the smaller type, in registers from the start, while tokens are counted.
template <typename T, typename O, bool TABLE, bool BACK>
__global__ __launch_bounds__(threads_of(TABLE)) void adjust_kernel(Adjust a, const typename T::raw *logits, const typename O::raw *grad,
                                                                   typename std::conditional<BACK, T, O>::type::raw *out)
{
    using W = typename std::conditional<BACK, T, O>::type;      // written
    using R = typename std::conditional<BACK, O, T>::type;      // read, column by column
    constexpr int VEC = T::VEC, THREADS = threads_of(TABLE), VECTORS = COLUMNS / VEC / THREADS;
    constexpr uint32_t ALL = (1u << VEC) - 1;
    extern __shared__ __align__(16) uint32_t table[];   // [COLUMNS], then the slice's biases
    __shared__ int32_t n_biases;
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x / a.slices;
    const int slice = (int)(blockIdx.x % a.slices);
    const typename T::raw *const x = logits + row * a.stride;
    const typename R::raw *from_row;
    if constexpr (BACK)
        from_row = grad + row * a.grad_stride;
    else
        from_row = x;
    typename W::raw *const y = out + row * a.out_stride;
    // Vectors are counted from the 16 bytes that the row begins in: the first and the last may be cut.
    const int off = (int)((reinterpret_cast<uintptr_t>(from_row) & 15) / sizeof(typename R::raw)) % VEC;
    const int vocab = (int)a.vocab, from = slice * COLUMNS - off;   // the slice's first column
    const gdp_adjust_history &h = a.history;
    Bias *const biases = reinterpret_cast<Bias *>(table + COLUMNS);
    constexpr int BIAS_WAVE = THREADS - 64;
    uint64_t token[HISTORY_AHEAD], bias_token = 0;
    int64_t length = 0, prompt = 0;
    float bias_value = 0.0f;
    const int64_t first = a.first + from;     // token of the slice's first column
    if constexpr (TABLE) {
        if (h.tokens) {
            length = at_most(h.lengths, h.length_type, row, h.places, h.places);
            prompt = at_most(h.prompts, h.prompt_type, row, 0, length);
            load_tokens<THREADS>(token, h.tokens, h.token_type, row * h.stride, t, length);
        }
        if constexpr (!BACK)
            if (t - BIAS_WAVE >= 0 && t - BIAS_WAVE < a.biases) {
                bias_token = (uint64_t)token_at(a.bias_tokens, a.bias_token_type, row * a.bias_stride + t - BIAS_WAVE);
                bias_value = a.bias[row * a.bias_stride + t - BIAS_WAVE];
            }
    }
    const float scale = a.scales ? a.scales[row] : a.scale;
    float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
    if (TABLE && h.tokens) {
        repetition = h.repetitions ? h.repetitions[row] : h.repetition;
        frequency = h.frequencies ? h.frequencies[row] : h.frequency;
        presence = h.presences ? h.presences[row] : h.presence;
    }
    // VEC bits of the mask for each vector, 0 outside of the row
    const uint32_t *const words = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    uint32_t mask[VECTORS];
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
        const int j = from + (u * THREADS + t) * VEC;
        const int skip = j < 0 ? -j : 0;
        uint32_t inside = j >= vocab ? 0 : ALL << skip & ALL;
        if (j + VEC > vocab && j < vocab) inside &= ALL >> (j + VEC - vocab);
        mask[u] = inside;
        if (words && inside) {
            const int64_t bit = a.first + j + skip, last = a.first + (j + VEC < vocab ? j + VEC : vocab) - 1;
            uint64_t w = words[bit >> 5];
            if (last >> 5 != bit >> 5) w |= (uint64_t)words[last >> 5] << 32;
            mask[u] = (uint32_t)(w >> (bit & 31)) << skip & inside;
        }
    }
    if constexpr (TABLE) {
#pragma unroll
        for (int i = 0; i < COLUMNS / 4 / THREADS; ++i) reinterpret_cast<uint4 *>(table)[i * THREADS + t] = make_uint4(0, 0, 0, 0);
        if (t == 0) n_biases = 0;
    }
    Pack<R, VEC> p[VECTORS];
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
        const int j = from + (u * THREADS + t) * VEC;
        if (j >= 0 && j + VEC <= vocab && mask[u] && !(a.in_place && mask[u] == ALL)) p[u].load(from_row + j);
    }
    if constexpr (TABLE) {
        __syncthreads();
        for (int64_t i = t; i < length;) {
#pragma unroll
            for (int u = 0; u < HISTORY_AHEAD; ++u) {
                const uint64_t local = token[u] - (uint64_t)first;
                if (i + u * THREADS >= length || local >= COLUMNS) continue;
                if (i + u * THREADS < prompt)
                    atomicOr(&table[local], OF_PROMPT);
                else
                    atomicAdd(&table[local], 1u);
            }
            i += THREADS * HISTORY_AHEAD;
            load_tokens<THREADS>(token, h.tokens, h.token_type, row * h.stride, i, length);
        }
        if constexpr (!BACK)
            if (a.biases && t >= BIAS_WAVE) {   // one wave, in order
                const int lane = t - BIAS_WAVE;
                int count = 0;
                for (int i = lane; i - lane < a.biases; i += 64) {
                    if (i >= 64 && i < a.biases) {
                        bias_token = (uint64_t)token_at(a.bias_tokens, a.bias_token_type, row * a.bias_stride + i);
                        bias_value = a.bias[row * a.bias_stride + i];
                    }
                    const uint64_t local = bias_token - (uint64_t)first;
                    const bool here = i < a.biases && local < COLUMNS;
                    const uint64_t all = __ballot(here);
                    if (here) {
                        biases[count + __popcll(all & ((1ull << lane) - 1))] = {(int32_t)local, bias_value};
                        atomicOr(&table[local], HAS_BIAS);
                    }
                    count += __popcll(all);
                }
                if (lane == 0) n_biases = count;
            }
        __syncthreads();
    }
    // Of a vector with tokens of the history or biases, and of what is not changed otherwise
    bool touched[VECTORS];
    Pack<T, VEC> sign[VECTORS];
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
        touched[u] = false;
        if constexpr (TABLE) {
            const uint4 *const c = reinterpret_cast<const uint4 *>(table + (u * THREADS + t) * VEC);
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < VEC / 4; ++i) any |= c[i].x | c[i].y | c[i].z | c[i].w;
            touched[u] = any != 0;
            const int j = from + (u * THREADS + t) * VEC;
            if (touched[u] && j >= 0 && j + VEC <= vocab) {
                if (a.in_place && mask[u] == ALL) p[u].load(from_row + j);
                if constexpr (BACK) sign[u].load(x + j);
            }
        }
    }
    // `of` is the logit by whose sign a repetition goes
    const auto of_column = [&](float f, float of, int local) -> float {
        if constexpr (TABLE) {
            const uint32_t c = table[local];
            if constexpr (BACK) f *= scale;
            if (c & (OF_PROMPT | COUNT)) f = of > 0.0f ? f / repetition : f * repetition;
            if constexpr (BACK) return f;
            if (c & COUNT) f = f - frequency * (float)(c & COUNT) - presence;
            if (c & HAS_BIAS) {
                float sum = 0.0f;
                for (int i = 0; i < n_biases; ++i) sum += biases[i].column == local ? biases[i].value : 0.0f;
                f += sum;
            }
        }
        return f * scale;
    };
    const float ruled_out = BACK ? 0.0f : -__builtin_inff();
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
        const int v = u * THREADS + t, j = from + v * VEC;
        if (j >= vocab) continue;
        if (j >= 0 && j + VEC <= vocab) {
            if (a.in_place && mask[u] == ALL && !touched[u]) continue;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = p[u][i] * scale;
            if (touched[u])
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    if constexpr (BACK)
                        f[i] = of_column(p[u][i], sign[u][i], v * VEC + i);
                    else
                        f[i] = of_column(p[u][i], p[u][i], v * VEC + i);
                }
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = mask[u] >> i & 1 ? f[i] : ruled_out;
            Pack<W, VEC> q;
            q.set(f);
            q.store(y + j);
        } else {
            for (int i = 0; i < VEC; ++i) {
                if (j + i < 0 || j + i >= vocab) continue;
                const bool allowed = mask[u] >> i & 1;
                if (a.in_place && allowed && (!TABLE || table[v * VEC + i] == 0)) continue;
                const float f = R::up(from_row[j + i]);
                y[j + i] = W::down(!allowed ? ruled_out : of_column(f, BACK && touched[u] ? T::up(x[j + i]) : f, v * VEC + i));
            }
        }
    }
}

// ---- host ----
constexpr int64_t MOST_ROWS = (int64_t)1 << 21, MOST_GROUPS = ((int64_t)1 << 23) - 1;   // a grid has less than 2^32 threads
bool token_aligned(const void *p, int type) { return aligned(p, type == GDP_I64 ? 8 : 4); }

int check(const gdp_adjust &a)
{
    if (a.n < 0 || a.vocab < 1 || a.first < 0) return gdp_fail(GDP_E_BADARG, "gdp_adjust: a size is negative, or there are no columns");
    if (a.n > MOST_ROWS || a.vocab > GDP_MAX_VOCAB || a.first > INT32_MAX - a.vocab)
        return gdp_fail(GDP_E_BADARG, "gdp_adjust: more than 2^21 rows or GDP_MAX_VOCAB columns, or a token above 2^31");
    if (!type_ok(a.logits_type) || !type_ok(a.out_type)) return gdp_fail(GDP_E_BADARG, "gdp_adjust: unknown element type");
    if (a.out_type != a.logits_type && a.out_type != GDP_F32) return gdp_fail(GDP_E_BADARG, "gdp_adjust: out_type must be that of the logits, or GDP_F32");
    const gdp_adjust_history &h = a.history;
    if (h.tokens) {
        if (h.places < 0 || h.places > MOST_PLACES) return gdp_fail(GDP_E_BADARG, "gdp_adjust: a history must have 0 to 2^30 - 1 places");
        if (!token_type_ok(h.token_type) || (h.lengths && !token_type_ok(h.length_type)) || (h.prompts && !token_type_ok(h.prompt_type)))
            return gdp_fail(GDP_E_BADARG, "gdp_adjust: unknown type of a history's numbers");
        if (!rows_ok(a.n, h.places, h.stride, false)) return gdp_fail(GDP_E_BADARG, "gdp_adjust: a history's stride is negative or too large");
        if (!token_aligned(h.tokens, h.token_type) || !token_aligned(h.lengths, h.length_type) || !token_aligned(h.prompts, h.prompt_type) ||
            !aligned(h.repetitions, 4) || !aligned(h.frequencies, 4) || !aligned(h.presences, 4))
            return gdp_fail(GDP_E_BADARG, "gdp_adjust: a pointer of the history is not aligned to its elements");
        if (!h.repetitions && !(h.repetition > 0.0f && h.repetition < 1e30f)) return gdp_fail(GDP_E_BADARG, "gdp_adjust: repetition must be positive and below 1e30");
        if ((!h.frequencies && !(h.frequency > -1e30f && h.frequency < 1e30f)) || (!h.presences && !(h.presence > -1e30f && h.presence < 1e30f)))
            return gdp_fail(GDP_E_BADARG, "gdp_adjust: frequency and presence must be between -1e30 and 1e30");
    }
    if (a.biases < 0 || a.biases > GDP_MAX_BIASES) return gdp_fail(GDP_E_BADARG, "gdp_adjust: biases must be 0 to GDP_MAX_BIASES");
    if (a.biases) {
        if (!a.bias_tokens || !a.bias) return gdp_fail(GDP_E_BADARG, "gdp_adjust: null pointer");
        if (!token_type_ok(a.bias_token_type)) return gdp_fail(GDP_E_BADARG, "gdp_adjust: unknown type of the biases' tokens");
        if (!token_aligned(a.bias_tokens, a.bias_token_type) || !aligned(a.bias, 4) || !rows_ok(a.n, a.biases, a.bias_stride, false))
            return gdp_fail(GDP_E_BADARG, "gdp_adjust: biases are not aligned to their elements, or their stride is negative or too large");
    }
    if (a.allowed) {
        if (a.words < (a.first + a.vocab + 31) / 32) return gdp_fail(GDP_E_BADARG, "gdp_adjust: the mask has fewer words than the vocabulary needs");
        if (!aligned(a.allowed, 4) || !rows_ok(a.n, a.words, a.allowed_stride, false))
            return gdp_fail(GDP_E_BADARG, "gdp_adjust: the mask is not aligned to its words, or its stride is negative or too large");
    }
    if (!aligned(a.scales, 4)) return gdp_fail(GDP_E_BADARG, "gdp_adjust: a pointer is not aligned to its elements");
    if (!a.scales && !(a.scale > 0.0f && a.scale < 1e30f)) return gdp_fail(GDP_E_BADARG, "gdp_adjust: scale must be positive and below 1e30");
    return GDP_OK;
}
int check_rows(const void *p, int64_t n, int64_t vocab, int64_t stride, int type, bool written)
{
    if (!p) return gdp_fail(GDP_E_BADARG, "gdp_adjust: null pointer");
    if (!rows_ok(n, vocab, stride, written)) return gdp_fail(GDP_E_BADARG, "gdp_adjust: a row stride is negative, too large, or below the width of rows that are written");
    return aligned(p, size_of(type)) ? GDP_OK : gdp_fail(GDP_E_BADARG, "gdp_adjust: a pointer is not aligned to its elements");
}

template <bool BACK> int run(const gdp_adjust &a, const void *grad, int64_t grad_stride, const char *who, void *stream)
{
    // Of the gradient only the repetition is of interest
    const bool history = a.history.tokens && a.history.places > 0, table = history || (!BACK && a.biases > 0);
    // one more vector where a row begins within 16 bytes
    const int64_t vec = 16 / size_of(a.logits_type), slices = ceil_div((ceil_div(a.vocab, vec) + 1) * vec, (int64_t)COLUMNS);
    if (a.n * slices > MOST_GROUPS) return gdp_fail(GDP_E_BADARG, "gdp_adjust: too many rows of so many columns");
    Adjust k{a.vocab, a.logits_stride, a.out_stride, grad_stride, a.first, (int32_t)slices, a.history, a.bias_tokens, a.bias,
             a.bias_stride, BACK ? 0 : a.biases, a.bias_token_type, a.allowed, a.allowed_stride, a.scales, a.scale, 0};
    if (!history) k.history.tokens = nullptr;
    k.in_place = a.out == (BACK ? grad : a.logits) && !a.scales && a.scale == 1.0f;
    const size_t lds = table ? COLUMNS * 4 + (size_t)k.biases * sizeof(Bias) : 0;
    return with_type(a.logits_type, [&](auto T) {
        using TT = decltype(T);
        const auto with = [&](auto O) {
            using OO = decltype(O);
            const auto *x = static_cast<const typename TT::raw *>(a.logits);
            const auto *g = static_cast<const typename OO::raw *>(grad);
            auto *y = static_cast<typename std::conditional<BACK, TT, OO>::type::raw *>(a.out);
            const dim3 grid((unsigned)(a.n * k.slices));
            return table ? launch(who, adjust_kernel<TT, OO, true, BACK>, grid, threads_of(true), lds, stream, k, x, g, y)
                         : launch(who, adjust_kernel<TT, OO, false, BACK>, grid, threads_of(false), 0, stream, k, x, g, y);
        };
        return a.out_type == GDP_F32 ? with(F32{}) : with(TT{});
    });
}

}  // namespace

extern "C" int gdp_adjust_forward(const gdp_adjust *a, void *stream)
{
    gdp_clear_error();
    if (!a) return gdp_fail(GDP_E_BADARG, "gdp_adjust: null argument");
    if (const int rc = check(*a)) return rc;
    if (a->n == 0) return GDP_OK;
    if (const int rc = check_rows(a->logits, a->n, a->vocab, a->logits_stride, a->logits_type, false)) return rc;
    if (const int rc = check_rows(a->out, a->n, a->vocab, a->out_stride, a->out_type, true)) return rc;
    if (a->out == a->logits && (a->out_type != a->logits_type || (a->n > 1 && a->out_stride != a->logits_stride)))
        return gdp_fail(GDP_E_BADARG, "gdp_adjust: a result in the place of the logits needs their type and stride");
    return run<false>(*a, nullptr, 0, "gdp_adjust_forward", stream);
}

extern "C" int gdp_adjust_backward(const gdp_adjust_grad *a, void *stream)
{
    gdp_clear_error();
    if (!a) return gdp_fail(GDP_E_BADARG, "gdp_adjust: null argument");
    const gdp_adjust &g = a->given;
    if (const int rc = check(g)) return rc;
    if (g.n == 0) return GDP_OK;
    if (g.history.tokens && g.history.places > 0)
        if (const int rc = check_rows(g.logits, g.n, g.vocab, g.logits_stride, g.logits_type, false)) return rc;
    if (const int rc = check_rows(a->grad, g.n, g.vocab, a->grad_stride, g.out_type, false)) return rc;
    if (const int rc = check_rows(g.out, g.n, g.vocab, g.out_stride, g.logits_type, true)) return rc;
    if (g.out == a->grad && (g.out_type != g.logits_type || (g.n > 1 && g.out_stride != a->grad_stride)))
        return gdp_fail(GDP_E_BADARG, "gdp_adjust: a gradient in the place of the other needs its type and stride");
    return run<true>(g, a->grad, a->grad_stride, "gdp_adjust_backward", stream);
}
