// Host side of the operators on logits (csrc/logit_*.hip) under AddressSanitizer and UndefinedBehaviorSanitizer, without a GPU: the sizes of
// workspaces, up to the largest that are permitted, and the checks of calls whose members are drawn from the ends of their ranges.
// Every call here is refused on the host, or has nothing to do: each has an argument that no check lets through, looked at last.
// Linked with the operators' own sources (host code instrumented); this program stands in for the library's error functions.
// Built and run by tests/test_sanitizers_logits.py.
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>

#include <hip/hip_runtime.h>

#include "../../include/galvatron_ops_hip.h"

void gdp_clear_error() {}
int gdp_fail(int code, const char *) { return code; }
int gdp_fail_hip(hipError_t, const char *what)
{
    fprintf(stderr, "logits_check: %s was launched\n", what);
    exit(1);
}

namespace {

unsigned long long rng_state = 0x9E3779B97F4A7C15ULL;
unsigned long long rnd()
{
    rng_state ^= rng_state << 13;
    rng_state ^= rng_state >> 7;
    rng_state ^= rng_state << 17;
    return rng_state;
}
template <typename T, size_t N> T one_of(const T (&v)[N]) { return v[rnd() % N]; }

int64_t size()
{
    static const int64_t ends[] = {INT64_MIN, -(1ll << 40), -1, 0, 1, 2, 3, 7, 8, 64, 255, 256, 257, 1024, 1025, 4096, 8191, 8192, 16383, 16384, 50257, 128256, (1 << 18) - 1, 1 << 18,
                                   (1 << 21) - 1, 1 << 21, (1 << 21) + 1, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, 1 << 29, (1 << 29) + 1, INT32_MAX - 1, INT32_MAX, 1ll << 31, 1ll << 58, 1ll << 59,
                                   INT64_MAX - 1, INT64_MAX};
    return rnd() % 2 ? one_of(ends) : (int64_t)(rnd() >> (rnd() % 64)) * (rnd() % 16 ? 1 : -1);
}
int32_t few() { static const int32_t v[] = {INT32_MIN, -1, 0, 0, 1, 1, 2, 2, 3, 64, 256, 257, 1024, INT32_MAX}; return one_of(v); }
float number() { static const float v[] = {-INFINITY, -1.0f, 0.0f, 1e-30f, 0.5f, 1.0f, 1.0f, 1e30f, INFINITY, NAN}; return one_of(v); }
template <typename T> T *place() { static const uintptr_t v[] = {0, 1, 2, 4, 8, 16, 256, 1 << 20, 1 << 20, 1 << 20, 1 << 20, UINTPTR_MAX}; return reinterpret_cast<T *>(one_of(v)); }
void *const ODD = reinterpret_cast<void *>(1);   // aligned to no element of more than a byte

int failures = 0, calls = 0;
void refused(int rc, bool nothing, const char *what)
{
    ++calls;
    if (rc == GDP_E_BADARG || (nothing && rc == GDP_OK)) return;
    fprintf(stderr, "logits_check: %s: %d\n", what, rc);
    ++failures;
}
void at_least(int rc, size_t got, double least, const char *what)
{
    ++calls;
    if (rc == GDP_E_BADARG || (rc == GDP_OK && (double)got >= least && (double)got < 1e15)) return;
    fprintf(stderr, "logits_check: %s: %d, %zu bytes for %g\n", what, rc, got, least);
    ++failures;
}

}  // namespace

int main()
{
    size_t bytes;
    int accepted = 0;
    for (int i = 0; i < 400000; ++i) {
        bytes = 0;
        const int64_t n = size(), vocab = size();
        int rc = gdp_distill_workspace(n, vocab, few(), few(), &bytes);
        accepted += rc == GDP_OK;
        at_least(rc, bytes, 0.0, "gdp_distill_workspace");
        const gdp_distill d{n, vocab, ODD, size(), few(), few(), few(), few(), place<void>(), place<float>(), place<void>(), number(), number(), few(), 0,
                            place<float>(), place<float>(), place<float>(), place<float>(), place<void>(), (size_t)size()};
        refused(gdp_distill_forward(&d, nullptr), n == 0, "gdp_distill_forward");
        const gdp_distill_part p{n, vocab, size(), ODD, size(), few(), few(), few(), few(), place<void>(), place<float>(), place<void>(), number(), 0,
                                 place<float>(), place<float>(), place<void>(), (size_t)size()};
        refused(gdp_distill_parts(&p, nullptr), n == 0, "gdp_distill_parts");
        const gdp_distill_joint j{n, vocab, few(), few(), few(), few(), place<void>(), place<float>(), place<void>(), number(), number(), few(), 0,
                                  place<float>(), static_cast<float *>(ODD), place<float>(), place<float>(), place<float>(), place<float>()};
        refused(gdp_distill_join(&j, nullptr), n == 0, "gdp_distill_join");
        const gdp_distill_grad g{n, vocab, size(), size(), place<void>(), size(), few(), few(), few(), few(), place<void>(), place<void>(), place<float>(),
                                 place<float>(), place<float>(), place<float>(), number(), 0, ODD, size()};
        refused(gdp_distill_backward(&g, nullptr), n == 0, "gdp_distill_backward");
        const gdp_adjust_history h{place<void>(), size(), size(), few(), few(), few(), number(), number(), number(), place<void>(), place<void>(), place<float>(),
                                   place<float>(), place<float>()};
        gdp_adjust a{n, vocab, size(), place<void>(), size(), few(), few(), h, place<void>(), place<float>(), size(), few(), few(), place<uint32_t>(), size(), size(),
                     place<float>(), number(), 0, ODD, size()};
        refused(gdp_adjust_forward(&a, nullptr), n == 0, "gdp_adjust_forward");
        const gdp_adjust_grad b{a, place<void>(), size()};
        refused(gdp_adjust_backward(&b, nullptr), n == 0, "gdp_adjust_backward");
    }
    // the largest that are permitted
    at_least(gdp_distill_workspace(1 << 21, GDP_MAX_VOCAB, GDP_F32, GDP_MAX_LISTED, &bytes), bytes, (double)(1 << 21) * (16 * 16 + 4 * 256), "most rows, widest");
    at_least(gdp_distill_workspace(1, GDP_MAX_VOCAB, GDP_BF16, 1, &bytes), bytes, 64.0 * 16 + 4, "one row, widest");
    if (failures || accepted < 1000) {
        fprintf(stderr, "logits_check: %d failures, %d sizes accepted\n", failures, accepted);
        return 1;
    }
    printf("logits_check: %d calls clean, %d sizes accepted\n", calls, accepted);
    return 0;
}
