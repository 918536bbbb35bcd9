// What the operators' translation units share: element types, rows of any alignment, sums over a wave, checks of calls.
#pragma once
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/galvatron_ops_hip.h"
#include "gdp_host.h"

namespace ops {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ---- element types: how a value is stored, and to and from float32 (rounding to nearest even) ----
struct F32 {
    using raw = uint32_t;
    static constexpr int VEC = 4;   // elements of 16 bytes
    static __device__ __forceinline__ float up(raw r) { return __builtin_bit_cast(float, r); }
    static __device__ __forceinline__ raw down(float f) { return __builtin_bit_cast(raw, f); }
};
struct F16 {
    using raw = uint16_t;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float up(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
    static __device__ __forceinline__ raw down(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
};
struct BF16 {
    using raw = uint16_t;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float up(raw r) { return __builtin_bit_cast(float, (uint32_t)r << 16); }
    static __device__ __forceinline__ raw down(float f) { return __builtin_bit_cast(raw, (__bf16)f); }
};

// Words in memory that are aligned to an element only.
template <int BYTES> struct Words;
template <> struct Words<2> {
    typedef uint32_t One __attribute__((aligned(2)));
    typedef uint32_t Two __attribute__((ext_vector_type(2), aligned(2)));
    typedef uint32_t Four __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct Words<4> {
    typedef uint32_t One __attribute__((aligned(4)));
    typedef uint32_t Two __attribute__((ext_vector_type(2), aligned(4)));
    typedef uint32_t Four __attribute__((ext_vector_type(4), aligned(4)));
};

// N neighbouring elements, read and written at once, wherever they begin: gfx950 takes addresses of any alignment, and a row that
// begins between words costs a second cache line for some lanes, not a read for each element.
template <typename T, int N> struct Pack {
    static constexpr int BYTES = N * (int)sizeof(typename T::raw);
    static constexpr int WORDS = BYTES >= 4 ? BYTES / 4 : 1;
    using One = typename Words<sizeof(typename T::raw)>::One;
    using Two = typename Words<sizeof(typename T::raw)>::Two;
    using Four = typename Words<sizeof(typename T::raw)>::Four;
    uint32_t w[WORDS];
    __device__ __forceinline__ typename T::raw raw(int i) const
    {
        if constexpr (sizeof(typename T::raw) == 4)
            return w[i];
        else
            return (typename T::raw)(w[i >> 1] >> (16 * (i & 1)));
    }
    __device__ __forceinline__ float operator[](int i) const { return T::up(raw(i)); }
    __device__ __forceinline__ void load(const typename T::raw *p)
    {
        if constexpr (BYTES == 2)
            w[0] = *p;
        else if constexpr (BYTES == 4)
            w[0] = *reinterpret_cast<const One *>(p);
        else if constexpr (BYTES == 8) {
            const Two v = *reinterpret_cast<const Two *>(p);
            w[0] = v.x, w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const Four v = reinterpret_cast<const Four *>(p)[i];
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        }
    }
    // ... of what is not read again: past the caches
    __device__ __forceinline__ void load_past(const typename T::raw *p)
    {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const Four v = __builtin_nontemporal_load(reinterpret_cast<const Four *>(p) + i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else
            load(p);
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void set(const float (&f)[N])
    {
        if constexpr (sizeof(typename T::raw) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = T::down(f[i]);
        } else if constexpr (N == 1) {
            w[0] = T::down(f[0]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) w[i] = (uint32_t)T::down(f[2 * i]) | ((uint32_t)T::down(f[2 * i + 1]) << 16);
        }
    }
    __device__ __forceinline__ void store(typename T::raw *p) const
    {
        if constexpr (BYTES == 2)
            *p = (typename T::raw)w[0];
        else if constexpr (BYTES == 4)
            *reinterpret_cast<One *>(p) = w[0];
        else if constexpr (BYTES == 8)
            *reinterpret_cast<Two *>(p) = Two{w[0], w[1]};
        else {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<Four *>(p)[i] = Four{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        }
    }
    // ... from element `from` on
    __device__ __forceinline__ void store_from(typename T::raw *p, int from) const
    {
        if (from == 0)
            store(p);
        else
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i >= from) p[i] = raw(i);
    }
    // ... of what is not read again soon: past the caches.  (Between fences for the compiler, which would make one store of this one and
    // an ordinary one on the other side of a branch.)
    __device__ __forceinline__ void store_past(typename T::raw *p) const
    {
        if constexpr (BYTES >= 16) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i)
                __builtin_nontemporal_store(Four{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]}, reinterpret_cast<Four *>(p) + i);
            asm volatile("" ::: "memory");
        } else
            store(p);
    }
};

// One element of a type that is known at run time (sums of columns, written once).
__device__ __forceinline__ void down_any(void *p, int type, int64_t at, float f)
{
    if (type == GDP_F32)
        static_cast<F32::raw *>(p)[at] = F32::down(f);
    else if (type == GDP_BF16)
        static_cast<BF16::raw *>(p)[at] = BF16::down(f);
    else
        static_cast<F16::raw *>(p)[at] = F16::down(f);
}

__device__ __forceinline__ int64_t token_at(const void *tokens, int type, int64_t i)
{
    return type == GDP_I64 ? static_cast<const int64_t *>(tokens)[i] : (int64_t) static_cast<const int32_t *>(tokens)[i];
}

// ---- over a wave of 64 ----
// DPP moves a value between lanes within an instruction: rows of 16 first, then the rows' last lanes on to the next rows; lane 63 has
// the result, which is read from there for all.  Lanes that have no source keep `idle`.
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ uint32_t dpp(uint32_t v, uint32_t idle)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)idle, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ float dpp(float v, float idle)
{
    return __builtin_bit_cast(float, dpp<CTRL, ROWS>(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, idle)));
}
constexpr int ROW_SHR1 = 0x111, ROW_SHR2 = 0x112, ROW_SHR4 = 0x114, ROW_SHR8 = 0x118, BCAST15 = 0x142, BCAST31 = 0x143;
constexpr int QUAD_SWAP1 = 0xB1, QUAD_SWAP2 = 0x4E;   // lanes 1 0 3 2, lanes 2 3 0 1

template <typename V, typename F> __device__ __forceinline__ V wave_fold(V v, V idle, F f)
{
    v = f(v, dpp<ROW_SHR1>(v, idle));
    v = f(v, dpp<ROW_SHR2>(v, idle));
    v = f(v, dpp<ROW_SHR4>(v, idle));
    v = f(v, dpp<ROW_SHR8>(v, idle));
    v = f(v, dpp<BCAST15, 0xa>(v, idle));
    v = f(v, dpp<BCAST31, 0xc>(v, idle));
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_sum(float v)
{
    return wave_fold(v, 0.0f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v)   // of what is no NaN
{
    return wave_fold(v, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    return wave_fold(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v)
{
    return wave_fold(v, ~0u, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v)
{
    return wave_fold(v, 0u, [](uint32_t a, uint32_t b) { return a + b; });
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // 1 ulp; below 2^-126: 0

__device__ __forceinline__ float finite_or_0(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// ---- host ----
template <typename F> int with_type(int t, F f)
{
    switch (t) {
    case GDP_F32: return f(F32{});
    case GDP_F16: return f(F16{});
    default: return f(BF16{});
    }
}
inline bool type_ok(int t) { return t == GDP_F32 || t == GDP_F16 || t == GDP_BF16; }
inline bool token_type_ok(int t) { return t == GDP_I32 || t == GDP_I64; }
inline int size_of(int t) { return t == GDP_F32 ? 4 : 2; }
inline bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline size_t round_up(size_t n, size_t to) { return (n + to - 1) / to * to; }
template <typename I> inline I ceil_div(I a, I b) { return (a + b - 1) / b; }
// Whether rows * stride + dim elements stay within what an offset in 64 bits can name, and rows do not overlap.
inline bool rows_ok(int64_t rows, int64_t dim, int64_t stride, bool written)
{
    return stride >= (written && rows > 1 ? dim : 0) && stride <= (INT64_MAX >> 4) / (rows > 0 ? rows : 1);
}
// Queues a kernel; GDP_OK or the launch's own error (an earlier one of the thread is neither reported nor cleared).
template <typename... P, typename... A>
inline int launch(const char *what, void (*kernel)(P...), dim3 grid, int threads, size_t lds, void *stream, A... given)
{
    const hipError_t e = [&](P... p) {
        void *args[] = {(void *)&p...};
        return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, dim3(threads), args, lds, static_cast<hipStream_t>(stream));
    }(given...);
    if (e == hipSuccess) return GDP_OK;
    (void)hipGetLastError();
    return gdp_fail_hip(e, what);
}

}  // namespace ops
