// Element types, unaligned vector access and cross-lane reductions shared by the operators that take device arrays of several
// types (experts.hip, distill.hip).
#pragma once
#include <exception>
#include <tuple>
#include "oak_internal.h"

namespace oak {

// Sums, softmax statistics and weights of T are held in Num<T>::acc: 32 bits for the 16- and 32-bit types, 64 for double.
template <typename T> struct Num { using acc = float; };
template <> struct Num<double> { using acc = double; };

// 16 bytes of T.  The alignment is the element's: rows may start anywhere (odd leading dimensions, sliced arrays) and gfx950's global
// loads and stores of 4 dwords need no more than that.
template <typename T> struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef T raw __attribute__((ext_vector_type(16 / sizeof(T))));
    typedef raw at __attribute__((aligned(sizeof(T))));
    static __device__ __forceinline__ raw load(const T* p) { return *reinterpret_cast<const at*>(p); }
    static __device__ __forceinline__ void store(T* p, raw v) { *reinterpret_cast<at*>(p) = v; }
    // results that no later kernel of the call reads: kept out of the caches' way
    static __device__ __forceinline__ void store_stream(T* p, raw v) { __builtin_nontemporal_store(v, reinterpret_cast<at*>(p)); }
};

inline size_t dtype_size(int dtype) { return dtype == OAK_F64 ? 8 : dtype == OAK_F32 ? 4 : 2; }
inline size_t dtype_acc_size(int dtype) { return dtype == OAK_F64 ? 8 : 4; }

// calls fn(T value) for the element type T of a run-time code
template <typename F> inline int with_dtype(int dtype, F&& fn) {
    switch (dtype) {
        case OAK_F64: return fn((double)0);
        case OAK_F32: return fn((float)0);
        case OAK_BF16: return fn((__bf16)0.0f);
        case OAK_F16: return fn((_Float16)0.0f);
        default: set_error("unknown element type %d", dtype); return OAK_E_ARG;
    }
}

// one value of an array whose type is only known at run time
__device__ __forceinline__ double load_any(const void* p, int dtype, int64_t i) {
    switch (dtype) {
        case OAK_F64: return static_cast<const double*>(p)[i];
        case OAK_F32: return (double)static_cast<const float*>(p)[i];
        case OAK_BF16: return (double)(float)static_cast<const __bf16*>(p)[i];
        default: return (double)(float)static_cast<const _Float16*>(p)[i];
    }
}

// ---- reductions over L consecutive lanes (L a power of two up to 64); every lane gets the result --------------------------
struct OpMax { template <typename A> __device__ __forceinline__ A operator()(A a, A b) const { return a > b ? a : b; } };
template <> __device__ __forceinline__ double OpMax::operator()(double a, double b) const { return __builtin_fmax(a, b); }
template <> __device__ __forceinline__ float OpMax::operator()(float a, float b) const { return __builtin_fmaxf(a, b); }
struct OpMin { template <typename A> __device__ __forceinline__ A operator()(A a, A b) const { return a < b ? a : b; } };
template <> __device__ __forceinline__ double OpMin::operator()(double a, double b) const { return __builtin_fmin(a, b); }
template <> __device__ __forceinline__ float OpMin::operator()(float a, float b) const { return __builtin_fminf(a, b); }
struct OpSum { template <typename A> __device__ __forceinline__ A operator()(A a, A b) const { return a + b; } };
struct OpOr { template <typename A> __device__ __forceinline__ A operator()(A a, A b) const { return a | b; } };

// The value of a lane in the other half of the block of 2 M lanes, M a constant power of two.  Within 16 lanes by a data-parallel
// move (a mirror of the block for M = 4 and 8: WHICH lane of the other half does not matter to a reduction that has already made
// each half agree), across rows of 16 and 32 by the row swaps -- none of it goes through LDS as a shuffle by index would.
template <int M> __device__ __forceinline__ unsigned lane_swap32(unsigned v) {
    if constexpr (M == 1) return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
    else if constexpr (M == 2) return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);   // quad_perm 2 3 0 1
    else if constexpr (M == 4) return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true);  // row_half_mirror
    else if constexpr (M == 8) return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true);  // row_mirror
    else {
        // both operands v: the first result holds the even rows (halves) twice, the second the odd ones
        const auto r = M == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        const unsigned lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
        return lane & M ? r[0] : r[1];
    }
}
template <int M, typename A> __device__ __forceinline__ A lane_swap(A v) {
    static_assert(sizeof(A) == 4 || sizeof(A) == 8, "32- and 64-bit values");
    if constexpr (sizeof(A) == 4) return __builtin_bit_cast(A, lane_swap32<M>(__builtin_bit_cast(unsigned, v)));
    else {
        const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
        return __builtin_bit_cast(A, (unsigned long long)lane_swap32<M>((unsigned)(b >> 32)) << 32 | lane_swap32<M>((unsigned)b));
    }
}

template <int L, typename Op, typename A> __device__ __forceinline__ A lanes_reduce(A v, Op op) {
    if constexpr (L > 1) v = op(v, lane_swap<1>(v));
    if constexpr (L > 2) v = op(v, lane_swap<2>(v));
    if constexpr (L > 4) v = op(v, lane_swap<4>(v));
    if constexpr (L > 8) v = op(v, lane_swap<8>(v));
    if constexpr (L > 16) v = op(v, lane_swap<16>(v));
    if constexpr (L > 32) v = op(v, lane_swap<32>(v));
    return v;
}

// exp(t), the float form as 2^(t log2 e) with log2 e in two parts (both positive: t = -inf gives 0)
__device__ __forceinline__ float exp_of(float t) { return __builtin_amdgcn_exp2f(__builtin_fmaf(t, 1.44269502162933349609f, t * 1.92596299112661e-8f)); }
// a b + c with c a constant of the code, read from scalar registers.  The compiler would rather have the constant in vector registers, where a
// polynomial's constants cost either a move per step or two registers each for as long as a loop lasts.
__device__ __forceinline__ double fma_const(double a, double b, double c) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
}
// Cody-Waite reduction and the Taylor polynomial of degree 13 on |r| <= ln 2 / 2 (remainder 4e-18), without the special cases of exp();
// beyond t = 709.8 infinite (t of at most 1e9, so that n fits 32 bits), NaN stays NaN
__device__ __forceinline__ double exp_of(double t) {
    t = t < -800.0 ? -800.0 : t;
    const double n = __builtin_rint(t * 1.4426950408889634074);
    const double r = __builtin_fma(n, -1.9082149292705877e-10, __builtin_fma(n, -6.93147180369123816490e-01, t));
    double p = fma_const(r, 1.0 / 6227020800.0, 1.0 / 479001600.0);
    p = fma_const(p, r, 1.0 / 39916800.0);
    p = fma_const(p, r, 1.0 / 3628800.0);
    p = fma_const(p, r, 1.0 / 362880.0);
    p = fma_const(p, r, 1.0 / 40320.0);
    p = fma_const(p, r, 1.0 / 5040.0);
    p = fma_const(p, r, 1.0 / 720.0);
    p = fma_const(p, r, 1.0 / 120.0);
    p = fma_const(p, r, 1.0 / 24.0);
    p = fma_const(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// 1 / d for normal d: the reciprocal's estimate and two Newton steps
__device__ __forceinline__ double inverse(double d) {
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}
__device__ __forceinline__ float inverse(float d) { return 1.0f / d; }
// log x for x >= 0 (log 0 = -inf, NaN stays NaN): x = 2^n m, m in [1/sqrt 2, sqrt 2), log m = 2 atanh f, f = (m - 1) / (m + 1), |f| < 0.172,
// by its series to f^21 (remainder 2e-18)
__device__ __forceinline__ double log_of(double x) {
    double m = __builtin_amdgcn_frexp_mant(x);
    int n = __builtin_amdgcn_frexp_exp(x);
    if (m < 0.70710678118654752440) { m *= 2.0; n -= 1; }
    const double f = (m - 1.0) * inverse(m + 1.0), s = f * f;
    double p = fma_const(s, 1.0 / 21.0, 1.0 / 19.0);
    p = fma_const(p, s, 1.0 / 17.0);
    p = fma_const(p, s, 1.0 / 15.0);
    p = fma_const(p, s, 1.0 / 13.0);
    p = fma_const(p, s, 1.0 / 11.0);
    p = fma_const(p, s, 1.0 / 9.0);
    p = fma_const(p, s, 1.0 / 7.0);
    p = fma_const(p, s, 1.0 / 5.0);
    p = fma_const(p, s, 1.0 / 3.0);
    const double two_f = f + f;
    const double r = __builtin_fma((double)n, 6.93147180369123816490e-01, __builtin_fma((double)n, 1.9082149292705877e-10, __builtin_fma(two_f * s, p, two_f)));
    return x == 0.0 ? -INFINITY : r;
}

// order of LDS accesses between the lanes of one wave (no other wave is waited for)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The launch's own status: hipGetLastError() would also report an error some other library of the process left behind.
template <typename... P, typename... A>
inline int launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t stream, A&&... args) {
    std::tuple<P...> held{static_cast<P>(args)...};
    void* ptrs[sizeof...(P)];
    int i = 0;
    std::apply([&](auto&... a) { ((ptrs[i++] = (void*)&a), ...); }, held);
    OAK_HIP_CHECK(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, ptrs, lds, stream));
    return OAK_OK;
}

// no C++ exception leaves a C entry point
template <typename F> inline int c_entry(F&& fn) {
    try { return fn(); }
    catch (const std::exception& e) { set_error("%s", e.what()); return OAK_E_HIP; }
    catch (...) { set_error("unknown C++ exception"); return OAK_E_HIP; }
}

// the device entry points run on the context's device and leave the thread's current one as it was
struct DeviceGuard {
    int before = -1; bool switched = false;
    int enter(const oak_ctx* ctx) {
        OAK_REQUIRE(ctx != nullptr, "ctx is NULL");
        OAK_HIP_CHECK(hipGetDevice(&before));
        if (before != ctx->device) { OAK_HIP_CHECK(hipSetDevice(ctx->device)); switched = true; }
        return OAK_OK;
    }
    ~DeviceGuard() { if (switched) (void)hipSetDevice(before); }
};

// host arrays of a call -> named scratch of the context and back.  Inputs are copied on the context's stream before the kernels,
// outputs behind them; finish() waits for that stream.
struct HostStage {
    oak_ctx* ctx;
    struct Out { void* host; void* dev; size_t bytes; };
    std::vector<Out> outs;
    explicit HostStage(oak_ctx* c) : ctx(c) {}
    template <typename P> int in(const char* name, P& p, size_t bytes) {
        if (p == nullptr || bytes == 0) return OAK_OK;
        void* d = nullptr;
        OAK_CHECK(get_buf(ctx, name, bytes, &d));
        OAK_HIP_CHECK(hipMemcpyAsync(d, p, bytes, hipMemcpyHostToDevice, ctx->stream));
        p = static_cast<P>(d);
        return OAK_OK;
    }
    template <typename P> int out(const char* name, P& p, size_t bytes) {
        if (p == nullptr || bytes == 0) return OAK_OK;
        void* d = nullptr;
        OAK_CHECK(get_buf(ctx, name, bytes, &d));
        outs.push_back({p, d, bytes});
        p = static_cast<P>(d);
        return OAK_OK;
    }
    int finish() {
        for (const Out& o : outs) OAK_HIP_CHECK(hipMemcpyAsync(o.host, o.dev, o.bytes, hipMemcpyDeviceToHost, ctx->stream));
        OAK_HIP_CHECK(hipStreamSynchronize(ctx->stream));
        return OAK_OK;
    }
};

}  // namespace oak
