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

constexpr int THREADS = 256;
constexpr int AHEAD = 4;                    // vectors that a thread has in flight
constexpr int HISTORY_AHEAD = 8;            // tokens
constexpr uint32_t OF_PROMPT = 1u << 31, HAS_BIAS = 1u << 30, COUNT = HAS_BIAS - 1;
constexpr int64_t MOST_PLACES = COUNT;      // of a history
constexpr int TABLE_COLUMNS = 8192;         // of a slice with a table: 32 KB of LDS, five workgroups on a core

struct Bias {
    int32_t column;      // of the slice
    float value;
};
struct Adjust {
    int64_t vocab, stride, out_stride, grad_stride, first;
    int32_t slices, width;   // vectors of a slice
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

// T: of the logits; O: of what is written, or of the gradient that is read (BACK).  TABLE: there is a history or are biases.
template <typename T, typename O, bool TABLE, bool BACK>
__global__ __launch_bounds__(THREADS) void adjust_kernel(Adjust a, const typename T::raw *logits, const typename O::raw *grad,
                                                         typename std::conditional<BACK, T, O>::type::raw *out)
{
    using W = typename std::conditional<BACK, T, O>::type;      // written
    using R = typename std::conditional<BACK, O, T>::type;      // read, column by column
    constexpr int VEC = T::VEC;
    extern __shared__ __align__(16) uint32_t table[];   // [width * VEC], then the slice's biases
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
    const int off = (int)((reinterpret_cast<uintptr_t>(from_row) & 15) / sizeof(typename R::raw)) % VEC;
    const int vocab = (int)a.vocab, vectors = (vocab + off + VEC - 1) / VEC;
    const int v0 = slice * a.width, v1 = v0 + a.width < vectors ? v0 + a.width : vectors;
    const int from = v0 * VEC - off, span = (v1 - v0) * VEC;     // the slice's first column (cut by the row), its columns
    const gdp_adjust_history &h = a.history;
    Bias *const biases = reinterpret_cast<Bias *>(table + a.width * VEC);
    if constexpr (TABLE) {
        for (int i = t; i < a.width * VEC / 4; i += THREADS) reinterpret_cast<uint4 *>(table)[i] = make_uint4(0, 0, 0, 0);
        if (t == 0) n_biases = 0;
        __syncthreads();
        if (h.tokens) {
            const int64_t length = at_most(h.lengths, h.length_type, row, h.places, h.places);
            const int64_t prompt = at_most(h.prompts, h.prompt_type, row, 0, length);
            const int64_t base_token = a.first + from;
            const uint64_t columns = span > 0 ? span : 0;
            const int64_t begin = row * h.stride;
            for (int64_t base = 0; base < length; base += THREADS * HISTORY_AHEAD) {
                uint64_t local[HISTORY_AHEAD];   // (of other slices, or none: above every column)
#pragma unroll
                for (int u = 0; u < HISTORY_AHEAD; ++u) {
                    const int64_t i = base + u * THREADS + t;
                    local[u] = i < length ? (uint64_t)token_at(h.tokens, h.token_type, begin + i) - (uint64_t)base_token : ~0ull;
                }
#pragma unroll
                for (int u = 0; u < HISTORY_AHEAD; ++u) {
                    if (local[u] >= columns) continue;
                    if (base + u * THREADS + t < prompt)
                        atomicOr(&table[local[u]], OF_PROMPT);
                    else
                        atomicAdd(&table[local[u]], 1u);
                }
            }
        }
        if constexpr (!BACK)
            if (a.biases && t < 64) {   // one wave, in order
                int count = 0;
                for (int base = 0; base < a.biases; base += 64) {
                    const int i = base + t;
                    uint64_t local = ~0ull;
                    float value = 0.0f;
                    if (i < a.biases) {
                        local = (uint64_t)token_at(a.bias_tokens, a.bias_token_type, row * a.bias_stride + i) - (uint64_t)(a.first + from);
                        value = a.bias[row * a.bias_stride + i];
                    }
                    const bool here = span > 0 && local < (uint64_t)span;
                    const uint64_t all = __ballot(here);
                    if (here) {
                        biases[count + __popcll(all & ((1ull << t) - 1))] = {(int32_t)local, value};
                        atomicOr(&table[local], HAS_BIAS);
                    }
                    count += __popcll(all);
                }
                if (t == 0) n_biases = count;
            }
        __syncthreads();
    }
    const float scale = a.scales ? a.scales[row] : a.scale;
    float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
    if (TABLE && h.tokens) {
        repetition = h.repetitions ? h.repetitions[row] : h.repetition;
        frequency = h.frequencies ? h.frequencies[row] : h.frequency;
        presence = h.presences ? h.presences[row] : h.presence;
    }
    const uint32_t *const words = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    const float ruled_out = BACK ? 0.0f : -__builtin_inff();
    // VEC bits of the mask, from column j on: the row's own columns only
    const auto allowed_of = [&](int j) -> uint32_t {
        constexpr uint32_t ALL = (1u << VEC) - 1;
        uint32_t inside = ALL;
        int skip = 0;
        if (j < 0) skip = -j, inside = ALL << skip & ALL;
        if (j + VEC > vocab) inside &= ALL >> (j + VEC - vocab);
        if (!words || !inside) return inside;
        const int64_t bit = a.first + j + skip;
        const int at = (int)(bit & 31);
        const int64_t last = a.first + (j + VEC < vocab ? j + VEC : vocab) - 1;
        uint64_t w = words[bit >> 5];
        if (last >> 5 != bit >> 5) w |= (uint64_t)words[last >> 5] << 32;
        return (uint32_t)(w >> at) << skip & inside;
    };
    const auto of_column = [&](float f, int local) -> float {   // local: of the slice
        if constexpr (TABLE) {
            const uint32_t c = table[local];
            if constexpr (BACK) {
                f *= scale;
                if (c & (OF_PROMPT | COUNT)) f = T::up(x[from + local]) > 0.0f ? f / repetition : f * repetition;
                return f;
            }
            if (c & (OF_PROMPT | COUNT)) f = f > 0.0f ? f / repetition : f * repetition;
            if (c & COUNT) f = f - frequency * (float)(c & COUNT) - presence;
            if (c & HAS_BIAS) {
                float sum = 0.0f;
                for (int i = 0; i < n_biases; ++i) sum += biases[i].column == local ? biases[i].value : 0.0f;
                f += sum;
            }
        }
        return f * scale;
    };
    for (int base = v0; base < v1; base += THREADS * AHEAD) {
        Pack<R, VEC> p[AHEAD];
        uint32_t mask[AHEAD];
        bool touched[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t;
            mask[u] = v < v1 ? allowed_of(v * VEC - off) : 0;
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            touched[u] = false;
            if constexpr (TABLE)
                if (v < v1) {
                    const uint4 *const c = reinterpret_cast<const uint4 *>(table + (v - v0) * VEC);
                    uint32_t any = 0;
#pragma unroll
                    for (int i = 0; i < VEC / 4; ++i) any |= c[i].x | c[i].y | c[i].z | c[i].w;
                    touched[u] = any != 0;
                }
            if (v < v1 && j >= 0 && j + VEC <= vocab && mask[u] && !(a.in_place && mask[u] == (1u << VEC) - 1 && !touched[u])) p[u].load(from_row + j);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int v = base + u * THREADS + t, j = v * VEC - off;
            if (v >= v1) continue;
            const bool whole = j >= 0 && j + VEC <= vocab;
            if (whole) {
                if (a.in_place && mask[u] == (1u << VEC) - 1 && !touched[u]) continue;
                float f[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = p[u][i] * scale;
                if (touched[u])
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f[i] = of_column(p[u][i], (v - v0) * VEC + i);
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = mask[u] >> i & 1 ? f[i] : ruled_out;
                Pack<W, VEC> q;
                q.set(f);
                q.store(y + j);
            } else {
                for (int i = 0; i < VEC; ++i)
                    if (j + i >= 0 && j + i < vocab && !(a.in_place && mask[u] >> i & 1 && (!TABLE || table[(v - v0) * VEC + i] == 0)))
                        y[j + i] = W::down(mask[u] >> i & 1 ? of_column(R::up(from_row[j + i]), (v - v0) * VEC + i) : ruled_out);
            }
        }
    }
}

// ---- host ----
constexpr int64_t MOST_ROWS = (int64_t)1 << 21, MOST_GROUPS = (int64_t)1 << 23;   // a grid has less than 2^32 threads
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
    const int vec = 16 / size_of(a.logits_type);
    const int64_t vectors = ceil_div(a.vocab, (int64_t)vec) + 1;   // one more where a row begins within 16 bytes
    // Slices of 8192 columns with a table, of two rounds of reads without, more where the grid would be too large.
    const int64_t columns = table ? TABLE_COLUMNS : 2 * THREADS * AHEAD * vec;
    const int64_t slices = ceil_div(vectors * vec, columns);
    const int64_t width = ceil_div(vectors, slices);
    if (a.n * slices > MOST_GROUPS) return gdp_fail(GDP_E_BADARG, "gdp_adjust: too many rows of so many columns");
    Adjust k{a.vocab, a.logits_stride, a.out_stride, grad_stride, a.first, (int32_t)ceil_div(vectors, width), (int32_t)width, a.history, a.bias_tokens, a.bias,
             a.bias_stride, BACK ? 0 : a.biases, a.bias_token_type, a.allowed, a.allowed_stride, a.scales, a.scale, 0};
    if (!history) k.history.tokens = nullptr;
    k.in_place = a.out == (BACK ? grad : a.logits) && !a.scales && a.scale == 1.0f;
    const size_t lds = table ? (size_t)width * vec * 4 + (size_t)k.biases * sizeof(Bias) : 0;
    return with_type(a.logits_type, [&](auto T) {
        using TT = decltype(T);
        const auto with = [&](auto O) {
            using OO = decltype(O);
            const auto *x = static_cast<const typename TT::raw *>(a.logits);
            const auto *g = static_cast<const typename OO::raw *>(grad);
            auto *y = static_cast<typename std::conditional<BACK, TT, OO>::type::raw *>(a.out);
            const dim3 grid((unsigned)(a.n * k.slices));
            return table ? launch(who, adjust_kernel<TT, OO, true, BACK>, grid, THREADS, lds, stream, k, x, g, y)
                         : launch(who, adjust_kernel<TT, OO, false, BACK>, grid, THREADS, 0, stream, k, x, g, y);
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
