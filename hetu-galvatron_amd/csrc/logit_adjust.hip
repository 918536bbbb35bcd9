// Penalties for repeated tokens, biases of single tokens, a grammar's mask and a temperature on rows of logits, and the gradient.
//
// A workgroup has a slice of a row's columns, in registers from the start.  Meanwhile it reads the row's history and counts the slice's
// tokens in a table in LDS: for each column a bit for a token of the prompt, one for a token with a bias, and below them how often the
// token is in what was drawn.  Counts are whole numbers, so the order in which atomics add them up does not show.  A bias has a lane of its own,
// which works its column out and writes it behind the others; where a token has several, each of their lanes adds up all of them in the
// order they are given.  The gradient needs two bits: whether a token is in the history and whether its logit is above 0, which is read
// where the token is met.
//
// Few steps wait for each other: history, mask and columns are read side by side, the table is waited for once.  (With the columns read after the table
// was made 1024 x 128256 bf16 with histories, biases and masks took 249 us, not 118; with the table looked up in a pass of its own 216.)
#include "ops_common.h"

#include <type_traits>

namespace {
using namespace ops;

constexpr int THREADS = 512;
constexpr int HISTORY_AHEAD = 1;            // reads of 16 bytes of the history that a thread has in flight
constexpr int64_t MOST_PLACES = 1 << 29, FEW_PLACES = (1 << 14) - 1;   // of a history; of one whose counts fit an entry of 16 bits

// What a workgroup knows of its columns' tokens.
enum Table { NONE, HALVES, WORDS, BITS };   // nothing; entries of 16 or 32 bits; two bits (the gradient)

typedef uint16_t TwoBytes __attribute__((aligned(1)));
struct Bias {
    int32_t column;      // of the slice
    float value;
};
struct Adjust {
    int64_t vocab, stride, out_stride, grad_stride, first;
    int32_t slices;          // of a row
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
    int32_t past;            // written past the caches
};

__device__ __forceinline__ int64_t at_most(const void *p, int type, int64_t row, int64_t otherwise, int64_t most)
{
    const int64_t n = p ? token_at(p, type, row) : otherwise;
    return n < 0 ? 0 : n > most ? most : n;
}

// Neighbouring tokens of a history, as they lie there: 16 bytes at once, at any address that a token may have.
struct Tokens {
    static constexpr int WORDS = 4;
    Words<4>::Four w;
    __device__ __forceinline__ void load(const uint32_t *p) { w = *reinterpret_cast<const Words<4>::Four *>(p); }
    // The column of the one in word i, of a slice whose first column has token `first`; above every column for one of none.
    __device__ __forceinline__ uint32_t column(int i, bool wide, uint32_t first) const { return wide && w[i | 1] != 0 ? ~0u : w[i] - first; }
};

constexpr int columns_of(int vec, int vectors) { return THREADS * vec * vectors; }
constexpr int bytes_of(Table table, int columns) { return table == HALVES ? 2 * columns : table == WORDS ? 4 * columns : table == BITS ? columns / 4 : 0; }

// Bound by memory where rows are many: 1024 x 128256 bf16 with histories of 1024, biases and masks 118 us, 0.55 GB at 4.6 TB/s, 103 of them without
// histories and biases; the gradient of 2048 rows 235 us, 1.09 GB at 4.6 TB/s and 0.1 GB of logits at the tokens' places.  128 x 50257 float32 with
// histories of 16384 17 us, 12 without: of small numbers, which are frequent, one slice counts most.  Few rows wait for memory twice:
// 16 x 128256 with histories of 2048 7 us.
// T: of the logits; O: of what is written, or of the gradient that is read (BACK).  VECTORS: of a thread, each of as many columns as 16 bytes of
// logits are.  PAST: read past the caches.
template <typename T, typename O, Table TABLE, bool BACK, int VECTORS, bool PAST>
__global__ __launch_bounds__(THREADS) void adjust_kernel(Adjust a, const typename T::raw *logits, const typename O::raw *grad,
                                                         typename std::conditional<BACK, T, O>::type::raw *out)
{
    using W = typename std::conditional<BACK, T, O>::type;      // written
    using R = typename std::conditional<BACK, O, T>::type;      // read, column by column
    constexpr int VEC = T::VEC, COLUMNS = columns_of(VEC, VECTORS), TABLE_WORDS = bytes_of(TABLE, COLUMNS) / 4;
    constexpr uint32_t ALL = (1u << VEC) - 1;
    constexpr int ENTRY = TABLE == HALVES ? 16 : 32;            // bits of a table's entry
    constexpr uint32_t OF_PROMPT = 1u << (ENTRY - 1), HAS_BIAS = 1u << (ENTRY - 2), COUNT = HAS_BIAS - 1;
    extern __shared__ __align__(16) uint32_t table[];           // then the slice's biases; BITS: in the history, then above 0
    __shared__ int32_t again;                                   // a token has several biases
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
    Bias *const biases = reinterpret_cast<Bias *>(table + TABLE_WORDS);
    const int64_t first = a.first + from;     // token of the slice's first column
    constexpr int BIASES = TABLE == HALVES || TABLE == WORDS ? GDP_MAX_BIASES / THREADS : 0;   // of each thread
    float bias_value[BIASES + 1], of_bias[BIASES + 1];   // of a column, and its logit
    int bias_column[BIASES + 1];                         // of the slice, or -1
    int length = 0, prompt = 0;               // in words of 32 bits
    const bool wide = h.token_type == GDP_I64;
    const uint32_t *history = nullptr;
    Tokens token[HISTORY_AHEAD];
    if constexpr (TABLE != NONE) {
        if (h.tokens) {
            length = (int)at_most(h.lengths, h.length_type, row, h.places, h.places);
            prompt = (int)at_most(h.prompts, h.prompt_type, row, 0, length) << wide;
            length <<= wide;
            history = static_cast<const uint32_t *>(h.tokens) + ((row * h.stride) << wide);
#pragma unroll
            for (int u = 0; u < HISTORY_AHEAD; ++u) {
                const int i = (u * THREADS + t) * Tokens::WORDS;
                if (i + Tokens::WORDS <= length) token[u].load(history + i);
            }
        }
#pragma unroll
        for (int b = 0; b < BIASES; ++b) {
            const int i = b * THREADS + t;
            bias_column[b] = -1;
            if (i < a.biases) {
                const uint64_t local = (uint64_t)token_at(a.bias_tokens, a.bias_token_type, row * a.bias_stride + i) - (uint64_t)first;
                bias_value[b] = a.bias[row * a.bias_stride + i];
                if (local < COLUMNS && from + (int)local >= 0 && from + (int)local < vocab) bias_column[b] = (int)local;
            }
        }
    }
    // VEC bits of the mask for each whole vector, from the byte or the two that hold them
    const uint8_t *const allowed = a.allowed ? reinterpret_cast<const uint8_t *>(a.allowed + row * a.allowed_stride) : nullptr;
    const auto bit_of = [&](int j) { return (uint32_t)a.first + (uint32_t)j; };
    uint32_t mask[VECTORS];
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
        const int j = from + (u * THREADS + t) * VEC;
        mask[u] = ALL;
        if (allowed && j >= 0 && j + VEC <= vocab) {
            const uint32_t bit = bit_of(j), shift = bit & 7;
            mask[u] = (shift + VEC > 8 ? (uint32_t)*reinterpret_cast<const TwoBytes *>(allowed + (bit >> 3)) : allowed[bit >> 3]) >> shift & ALL;
        }
    }
    if constexpr (TABLE != NONE) {
#pragma unroll
        for (int i = t; i < TABLE_WORDS / 4; i += THREADS) reinterpret_cast<uint4 *>(table)[i] = make_uint4(0, 0, 0, 0);
        if (t == 0) again = 0;
    }
    Pack<R, VEC> p[VECTORS];
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
        const int j = from + (u * THREADS + t) * VEC;
        // With a table without waiting for the mask
        if (j >= 0 && j + VEC <= vocab && (TABLE != NONE ? !a.in_place : mask[u] && !(a.in_place && mask[u] == ALL))) {
            if constexpr (PAST)
                p[u].load_past(from_row + j);
            else
                p[u].load(from_row + j);
        }
    }
    const float scale = a.scales ? a.scales[row] : a.scale;
    float repetition = 1.0f, inverse = 1.0f, frequency = 0.0f, presence = 0.0f;
    if constexpr (TABLE != NONE) {
        if (h.tokens) {
            repetition = h.repetitions ? h.repetitions[row] : h.repetition;
            inverse = 1.0f / repetition;
            frequency = h.frequencies ? h.frequencies[row] : h.frequency;
            presence = h.presences ? h.presences[row] : h.presence;
        }
        __syncthreads();
        // N tokens' columns; those of other slices, or of none, are above all.  The first `of_prompt` are of the prompt.
        const auto count = [&](auto N, const uint32_t *column, int of_prompt) {
            if constexpr (TABLE == BITS) {
                bool positive[N.value], fresh[N.value];
#pragma unroll
                for (int k = 0; k < N.value; ++k) {
                    const int j = from + (int)column[k];
                    // (once is enough for a token that is there often)
                    fresh[k] = column[k] < COLUMNS && j >= 0 && j < vocab && !(table[column[k] >> 5] >> (column[k] & 31) & 1);
                    positive[k] = fresh[k] && T::up(x[j]) > 0.0f;
                }
#pragma unroll
                for (int k = 0; k < N.value; ++k)
                    if (fresh[k]) {
                        atomicOr(&table[column[k] >> 5], 1u << (column[k] & 31));
                        if (positive[k]) atomicOr(&table[TABLE_WORDS / 2 + (column[k] >> 5)], 1u << (column[k] & 31));
                    }
            } else {
#pragma unroll
                for (int k = 0; k < N.value; ++k)
                    if (column[k] < COLUMNS) {
                        uint32_t *const at = &table[TABLE == HALVES ? column[k] >> 1 : column[k]];
                        const int shift = TABLE == HALVES ? (column[k] & 1) * 16 : 0;
                        if (k < of_prompt)
                            atomicOr(at, OF_PROMPT << shift);
                        else
                            atomicAdd(at, 1u << shift);
                    }
            }
        };
        const int of_wave = __builtin_amdgcn_readfirstlane(t) * Tokens::WORDS;
        for (int base = 0; base < length; base += THREADS * HISTORY_AHEAD * Tokens::WORDS) {
#pragma unroll
            for (int u = 0; u < HISTORY_AHEAD; ++u) {
                const int i = base + (u * THREADS + t) * Tokens::WORDS;
                if (i + Tokens::WORDS <= length) {
                    uint32_t column[Tokens::WORDS];
#pragma unroll
                    for (int k = 0; k < Tokens::WORDS; ++k) column[k] = wide && k % 2 != 0 ? ~0u : token[u].column(k, wide, (uint32_t)first);
                    // (most waves' tokens are all of the prompt or all drawn)
                    constexpr std::integral_constant<int, Tokens::WORDS> N;
                    const int at = base + u * THREADS * Tokens::WORDS + of_wave;
                    if (at >= prompt)
                        count(N, column, 0);
                    else if (at + 64 * Tokens::WORDS <= prompt)
                        count(N, column, Tokens::WORDS);
                    else
                        count(N, column, prompt - i);
                } else {   // the last, one by one
                    for (int k = i; k < length; k += 1 + wide) {
                        const uint32_t column = wide && history[k + 1] != 0 ? ~0u : history[k] - (uint32_t)first;
                        count(std::integral_constant<int, 1>{}, &column, prompt - k);
                    }
                }
                const int next = i + THREADS * HISTORY_AHEAD * Tokens::WORDS;
                if (next + Tokens::WORDS <= length) token[u].load(history + next);
            }
        }
#pragma unroll
        for (int b = 0; b < BIASES; ++b)
            if (b * THREADS + t < a.biases) {
                const int column = bias_column[b];
                biases[b * THREADS + t] = {column, bias_value[b]};
                if (column < 0) continue;
                of_bias[b] = T::up(x[from + column]);   // (before anything is written)
                const int shift = TABLE == HALVES ? (column & 1) * 16 : 0;
                if (atomicOr(&table[TABLE == HALVES ? column >> 1 : column], HAS_BIAS << shift) >> shift & HAS_BIAS) again = 1;
            }
        __syncthreads();
    }
    // pen(f) less frequency and presence
    const auto penalised = [&](float f, uint32_t entry) -> float {
        const uint32_t n = entry & COUNT;
        f *= entry & (OF_PROMPT | COUNT) ? f > 0.0f ? inverse : repetition : 1.0f;
        return n ? fmaf(-frequency, (float)n, f) - presence : f;
    };
    // The results of columns with biases, which are written behind the others
#pragma unroll
    for (int b = 0; b < BIASES; ++b)
        if (bias_column[b] >= 0) {
            const int column = bias_column[b];
            if (again) {   // all that its token has, in their order, at each of them
                bias_value[b] = 0.0f;
                for (int i = 0; i < a.biases; ++i) bias_value[b] += biases[i].column == column ? biases[i].value : 0.0f;
            }
            const uint32_t entry = TABLE == HALVES ? table[column >> 1] >> (column & 1) * 16 & 0xffff : table[column];
            of_bias[b] = (penalised(of_bias[b], entry) + bias_value[b]) * scale;
            const uint32_t bit = bit_of(from + column);
            if (allowed && !(allowed[bit >> 3] >> (bit & 7) & 1)) bias_column[b] = -1;
        }
    if constexpr (BIASES > 0)
        if (a.biases && static_cast<const void *>(out) == logits) __syncthreads();   // (their logits are overwritten below)
    constexpr uint32_t RULED_OUT = BACK ? 0u : 0xff800000u;   // 0, -inf
#pragma unroll
    for (int u = 0; u < VECTORS; ++u) {
        const int v = u * THREADS + t, j = from + v * VEC;
        if (j >= vocab) continue;
        // the vector's entries
        uint32_t c[TABLE == BITS ? 2 : VEC * ENTRY / 32], any = 0;
        if constexpr (TABLE == BITS) {
            const uint8_t *const bytes = reinterpret_cast<const uint8_t *>(table);
            const int at = VEC == 8 ? v : v >> 1, shift = VEC == 8 ? 0 : 4 * (v & 1);
            any = c[0] = bytes[at] >> shift & ALL;
            c[1] = bytes[TABLE_WORDS * 2 + at] >> shift;
        } else if constexpr (TABLE != NONE) {
            Pack<F32, VEC * ENTRY / 32> entries;
            entries.load(table + v * (VEC * ENTRY / 32));
#pragma unroll
            for (int i = 0; i < VEC * ENTRY / 32; ++i) any |= c[i] = entries.w[i];
        }
        const auto of_column = [&](float f, int i) -> float {
            if constexpr (TABLE == BITS) {
                f *= scale;
                return c[0] >> i & 1 ? f * (c[1] >> i & 1 ? inverse : repetition) : f;
            }
            if constexpr (TABLE == HALVES || TABLE == WORDS) f = penalised(f, TABLE == HALVES ? c[i / 2] >> (i % 2) * 16 & 0xffff : c[i]);
            return f * scale;
        };
        if (j >= 0 && j + VEC <= vocab) {
            if (a.in_place) {
                if (mask[u] == ALL && !any) continue;
                if (TABLE != NONE) p[u].load(from_row + j);
            }
            float f[VEC];
            if (any) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = of_column(p[u][i], i);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = p[u][i] * scale;
            }
            if (allowed)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const uint32_t keep = (uint32_t)((int32_t)(mask[u] << (31 - i)) >> 31);
                    f[i] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, f[i]) & keep) | (RULED_OUT & ~keep));
                }
            Pack<W, VEC> q;
            q.set(f);
            if (a.past)
                q.store_past(y + j);
            else
                q.store(y + j);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (j + i < 0 || j + i >= vocab) continue;
                const bool keep = !allowed || allowed[bit_of(j + i) >> 3] >> (bit_of(j + i) & 7) & 1;
                if (a.in_place && keep && !any) continue;
                y[j + i] = W::down(keep ? of_column(R::up(from_row[j + i]), i) : __builtin_bit_cast(float, RULED_OUT));
            }
        }
    }
    if (BIASES && a.biases) {
        __syncthreads();
#pragma unroll
        for (int b = 0; b < BIASES; ++b)
            if (bias_column[b] >= 0) y[from + bias_column[b]] = W::down(of_bias[b]);
    }
}

// ---- host ----
// The last of the caches has 256 MB.  What does not fit it is read past the caches, results of half as much are written past them: the gradient of
// 2048 x 128256 bf16 252 us with neither, 243 with the result and 226 with both past the caches; forward 1024 x 128256 115 us, 107 with the result
// past them.  What fits is left to who reads it next.
constexpr int64_t READ_PAST = 256 << 20, WRITE_PAST = 128 << 20;
// Entries of 16 bits for histories whose counts they hold leave a core twice the columns: with entries of 32 bits and half the columns to a workgroup
// 1024 x 128256 with histories of 1024 147 us, not 133 (by graphs replayed after a wait, up to a tenth longer than on a busy
// device, as the rest was measured).  One read of the history in flight: with four, for which 64 registers are exceeded, 120 us there, not 107,
// and at 128 x 50257 float32 with all of 16384 places used 33 us, not 28.
// Four vectors a thread where that leaves no core without a workgroup, else one: 16 x 128256 bf16 with histories of 2048 12.2 us with four and 8.0
// with one, 77 x 32003 float32 (gradient) 10.6 and 11.8.
// Entries of 32 bits are built for four alone, few rows or many, and chosen by the places that a history has, not by those that count.  That leaves cores idle:
// one row of 128256 bf16 with a history of 16383 places 9.2 us, of 16384 11.1, of 32768 16.3; 16 rows 11.3, 11.9 and 22; where 1000 of the places count
// one row takes 5 us with 16383 of them and 7 with 32768.
constexpr int64_t CORES = 256;
// Slices of a row; one more vector where it begins within 16 bytes.
constexpr int64_t slices_of(int64_t vocab, int vec, int columns) { return ((vocab + vec - 1) / vec * vec + vec + columns - 1) / columns; }
constexpr int64_t MOST_ROWS = (int64_t)1 << 21, MOST_GROUPS = UINT32_MAX / THREADS;   // a grid has less than 2^32 threads
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
        if (h.places < 0 || h.places > MOST_PLACES) return gdp_fail(GDP_E_BADARG, "gdp_adjust: a history must have 0 to 2^29 places");
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
    const bool history = a.history.tokens && a.history.places > 0;
    Adjust k{a.vocab, a.logits_stride, a.out_stride, grad_stride, a.first, 0, a.history, a.bias_tokens, a.bias, a.bias_stride, BACK ? 0 : a.biases,
             a.bias_token_type, a.allowed, a.allowed_stride, a.scales, a.scale, 0, 0};
    if (!history) k.history.tokens = nullptr;
    k.past = a.n * a.vocab * size_of(BACK ? a.logits_type : a.out_type) >= WRITE_PAST;
    k.in_place = a.out == (BACK ? grad : a.logits) && !a.scales && a.scale == 1.0f;
    return with_type(a.logits_type, [&](auto T) {
        using TT = decltype(T);
        const auto with = [&](auto O) {
            using OO = decltype(O);
            const auto go = [&](auto TABLE, auto VECTORS, auto PAST) {
                constexpr int columns = columns_of(TT::VEC, VECTORS.value);
                const int64_t slices = slices_of(a.vocab, TT::VEC, columns);
                if (a.n * slices > MOST_GROUPS) return gdp_fail(GDP_E_BADARG, "gdp_adjust: too many rows of so many columns");
                k.slices = (int32_t)slices;
                return launch(who, adjust_kernel<TT, OO, TABLE.value, BACK, VECTORS.value, PAST.value>, dim3((unsigned)(a.n * slices)), THREADS,
                              (size_t)bytes_of(TABLE.value, columns) + (size_t)k.biases * sizeof(Bias), stream, k,
                              static_cast<const typename TT::raw *>(a.logits), static_cast<const typename OO::raw *>(grad),
                              static_cast<typename std::conditional<BACK, TT, OO>::type::raw *>(a.out));
            };
            const auto of_four = [&](auto TABLE) {
                const std::integral_constant<int, 4> four;
                return a.n * a.vocab * (int)sizeof(typename std::conditional<BACK, OO, TT>::type::raw) >= READ_PAST ? go(TABLE, four, std::true_type{})
                                                                                                                    : go(TABLE, four, std::false_type{});
            };
            const auto of_size = [&](auto TABLE) {
                return a.n * slices_of(a.vocab, TT::VEC, columns_of(TT::VEC, 4)) < CORES ? go(TABLE, std::integral_constant<int, 1>{}, std::false_type{})
                                                                                         : of_four(TABLE);
            };
            if constexpr (BACK)
                return history ? of_size(std::integral_constant<Table, BITS>{}) : of_size(std::integral_constant<Table, NONE>{});
            else {
                if (!history && !a.biases) return of_size(std::integral_constant<Table, NONE>{});
                return a.history.places <= FEW_PLACES || !history ? of_size(std::integral_constant<Table, HALVES>{})
                                                                  : of_four(std::integral_constant<Table, WORDS>{});
            }
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
