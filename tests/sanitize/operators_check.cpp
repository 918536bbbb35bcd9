// Host side of the operators (csrc/ops_*.hip) under AddressSanitizer and UndefinedBehaviorSanitizer, without a GPU: the sizes of their
// workspaces, up to the largest that are permitted, and their checks of calls whose members are drawn from the ends of their ranges.
// Every call here is refused on the host, or has nothing to do: each has an argument that no check lets through, looked at last, so that what
// is computed of the others before has run.  Linked with the operators' own sources (host code instrumented); this program stands
// in for the library's error functions.  Built and run by tests/test_sanitizers_operators.py.
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include <hip/hip_runtime.h>

#include "../../include/galvatron_ops_hip.h"

void gdp_clear_error() {}
int gdp_fail(int code, const char *) { return code; }
int gdp_fail_hip(hipError_t, const char *what)
{
    fprintf(stderr, "operators_check: %s was launched\n", what);
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
    static const int64_t ends[] = {INT64_MIN, INT64_MIN + 1, -(1ll << 40), -1, 0, 1, 2, 3, 7, 8, 63, 64, 65, 511, 512, 1023, 4095, 4096, 4097, 8192, 16383, 16384, 16385, 50257, 128256,
                                   (1 << 20) - 1, 1 << 20, (1 << 20) + 1, 1 << 21, (1 << 21) + 1, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, (1 << 26) - 4096, (1 << 26) - 4095, 1 << 27, (1 << 27) + 1, INT32_MAX - 1,
                                   INT32_MAX, 1ll << 31, 1ll << 32, 1ll << 58, 1ll << 59, INT64_MAX - 1, INT64_MAX};
    return rnd() % 2 ? one_of(ends) : (int64_t)(rnd() >> (rnd() % 64)) * (rnd() % 16 ? 1 : -1);
}
int32_t few() { static const int32_t v[] = {INT32_MIN, -1, 0, 0, 1, 1, 2, 2, 3, 63, 64, 65, INT32_MAX}; return one_of(v); }
float number() { static const float v[] = {-INFINITY, -1.0f, 0.0f, 1e-30f, 1.0f, 1.0f, 1.0f, 1e30f, INFINITY, NAN}; return one_of(v); }
void *place() { static const uintptr_t v[] = {0, 1, 2, 4, 8, 16, 256, 1 << 20, 1 << 20, 1 << 20, 1 << 20, UINTPTR_MAX}; return reinterpret_cast<void *>(one_of(v)); }
void *const ODD = reinterpret_cast<void *>(1);   // aligned to no element of more than a byte
gdp_norm_params side() { return {few(), few(), number(), 0, place(), place()}; }

int failures = 0, calls = 0;
void refused(int rc, bool nothing, const char *what)
{
    ++calls;
    if (rc == GDP_E_BADARG || (nothing && rc == GDP_OK)) return;
    fprintf(stderr, "operators_check: %s: %d\n", what, rc);
    ++failures;
}
void at_least(int rc, size_t got, double least, const char *what)
{
    ++calls;
    if (rc == GDP_E_BADARG || (rc == GDP_OK && (double)got >= least && (double)got < 1e15)) return;
    fprintf(stderr, "operators_check: %s: %d, %zu bytes for %g\n", what, rc, got, least);
    ++failures;
}

}  // namespace

int main()
{
    size_t bytes;
    int accepted = 0;
    for (int i = 0; i < 400000; ++i) {
        bytes = 0;
        int64_t n = size(), rows = size(), dim = size();
        int rc = gdp_embed_grad_workspace(n, rows, dim, &bytes);
        accepted += rc == GDP_OK;
        at_least(rc, bytes, rc ? 0.0 : 8.0 * n + 8.0 * rows + n / 128 * 8.0 * dim, "gdp_embed_grad_workspace");
        rc = gdp_logprob_workspace(n, dim, few(), few(), &bytes);
        accepted += rc == GDP_OK;
        at_least(rc, rc ? 0 : bytes, 0.0, "gdp_logprob_workspace");
        const int64_t gates = rnd() % 4 ? (int64_t)(rnd() % 5) : size();
        rc = gdp_norm_grad_workspace(n, dim, gates, &bytes);
        accepted += rc == GDP_OK;
        at_least(rc, bytes, rc || n == 0 ? 0.0 : 20.0 * dim, "gdp_norm_grad_workspace");

        const gdp_embed e{n, rows, dim, size(), ODD, few(), few(), few(), number(), place(), size(), place(), size()};
        refused(gdp_embed_forward(&e, nullptr), n == 0 || dim == 0, "gdp_embed_forward");
        const gdp_embed_grad eg{n, rows, dim, rnd() % 2 ? 0 : size(), place(), few(), few(), few(), few(), number(), place(), size(), place(), size(), place(), 0};
        refused(gdp_embed_backward(&eg, nullptr), rows == 0 || dim == 0 || n == 0, "gdp_embed_backward");
        const gdp_logprob l{n, dim, place(), size(), few(), few(), place(), number(), few(), nullptr, nullptr, nullptr, nullptr, nullptr, place(), (size_t)size()};
        refused(gdp_logprob_forward(&l, nullptr), n == 0, "gdp_logprob_forward");
        const gdp_logprob_stats ls{l, static_cast<float *>(place())};
        refused(gdp_logprob_forward_stats(&ls, nullptr), n == 0, "gdp_logprob_forward_stats");
        const gdp_logprob_part lp{n, dim, size(), place(), size(), few(), few(), place(), number(), few(), nullptr, nullptr, nullptr, place(), (size_t)size()};
        refused(gdp_logprob_parts(&lp, nullptr), n == 0, "gdp_logprob_parts");
        const gdp_logprob_joint_stats j{{n, dim, few(), few(), number(), few(), ODD, static_cast<float *>(place()), static_cast<float *>(place()), static_cast<int32_t *>(place()),
                                         static_cast<float *>(place()), static_cast<float *>(place()), static_cast<float *>(place()), static_cast<float *>(place()), static_cast<int64_t *>(place())},
                                        static_cast<float *>(place())};
        refused(gdp_logprob_join(&j.given, nullptr), n == 0, "gdp_logprob_join");
        refused(gdp_logprob_join_stats(&j, nullptr), n == 0, "gdp_logprob_join_stats");
        const gdp_logprob_grad_stats lg{{n, dim, size(), size(), place(), size(), few(), few(), place(), number(), few(), nullptr, nullptr, nullptr, nullptr,
                                         static_cast<float *>(place()), nullptr, nullptr, place(), size()}, static_cast<float *>(place())};   // one gradient of an entropy that is not there, or none
        refused(gdp_logprob_backward(&lg.given, nullptr), n == 0, "gdp_logprob_backward");
        gdp_logprob_grad_stats half = lg;
        half.given.grad_entropy = static_cast<float *>(ODD);
        refused(gdp_logprob_backward_stats(&half, nullptr), n == 0, "gdp_logprob_backward_stats");
        const gdp_norm no{n, dim, few(), few(), place(), size(), place(), size(), side(), side(), place(), gates, size(), few(), number(), number(), 0, place(), size(), place(), size(),
                          reinterpret_cast<float *>(4)};
        refused(gdp_norm_forward(&no, nullptr), n == 0, "gdp_norm_forward");
        const gdp_norm_grad ng{n, dim, few(), few(), place(), size(), place(), size(), static_cast<float *>(place()), place(), size(), place(), size(), side(), side(), place(), gates, size(), few(),
                               number(), number(), 0, place(), size(), place(), size(), nullptr, nullptr, nullptr, nullptr, nullptr, place(), 0};
        refused(gdp_norm_backward(&ng, nullptr), n == 0, "gdp_norm_backward");
    }
    // the largest that are permitted
    at_least(gdp_embed_grad_workspace((1 << 26) - 4096, 1 << 27, 1 << 20, &bytes), bytes, 4e12, "embedding, largest");
    at_least(gdp_logprob_workspace(1, GDP_MAX_VOCAB, GDP_F32, GDP_MAX_TOP, &bytes), bytes, 64.0 * (16 + 8 * 64), "log probabilities, widest");
    at_least(gdp_logprob_workspace(1 << 21, GDP_MAX_VOCAB, GDP_BF16, 0, &bytes), bytes, 0.0, "log probabilities, most rows");
    at_least(gdp_norm_grad_workspace((1 << 22) - 1, GDP_MAX_NORM_DIM, 0, &bytes), bytes, 20.0 * GDP_MAX_NORM_DIM, "norms, largest");
    if (failures || accepted < 1000) {
        fprintf(stderr, "operators_check: %d failures, %d sizes accepted\n", failures, accepted);
        return 1;
    }
    printf("operators_check: %d calls clean, %d sizes accepted\n", calls, accepted);
    return 0;
}
