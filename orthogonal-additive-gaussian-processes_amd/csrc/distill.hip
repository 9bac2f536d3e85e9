// Divergence of a student's class distribution from a teacher's top logits, and its gradient.
//
// With z = log sum_v exp(s_v / tau), q_v = exp(s_v / tau - z), "top" the teacher's entries and "rest" every other class:
//   forward  L = tau^2 w [ sum p_k (log p_k - log q_k) + p_r (log p_r - log q_r) ]
//            dL/ds_v = tau w (q_v - p_v) on the top,  tau w q_v (1 - p_r / q_r) on the rest   (p_r = 0 without a rest outcome)
//   reverse  L = tau^2 w [ sum q_k (log q_k - log p_k) + q_r (log q_r - log p_r) ]
//            dL/ds_v = tau w q_v (log q_b - log p_b - L / (tau^2 w)),  b the outcome v belongs to
// so the gradient is one coefficient times q_v on the rest and k values of their own on the top.
//
// q_r is summed over the rest itself (its own running maximum, the teacher's entries left out by a bit per class in LDS): taken
// as 1 - sum q_k it would lose every digit where the student is sure of itself.  The sums over the classes run in 32 bits (64 for
// double), everything per entry and per row in 64.
#include "lowp.h"

namespace oak {

struct DistillDev {
    int64_t n, ld, ld_top, ld_index, ld_out;
    int V, K, top_dtype, lse_dtype, weight_dtype, index_64, reverse;
    double tau, inv_tau, floor_rest;
    float c_hi, c_lo;           // log2(e) / tau in two floats, c_hi rounded towards zero
    const void* logits; const void* top; const void* index; const void* lse; const void* weight;
    void* loss; void* dlogits;
};

// exp(t / tau) for t <= 0.  float: 2^(t c) with c in two parts, since a c off by half a unit would put a common relative error of |t| c 2^-25
// on all the terms of a sum (t = 20: 1e-6 in log z, more than a small divergence bears).  Both parts are positive: t = -inf gives 0, NaN stays NaN.
__device__ __forceinline__ float exp_scaled(const DistillDev& a, float t) { return __builtin_amdgcn_exp2f(__builtin_fmaf(t, a.c_hi, t * a.c_lo)); }
__device__ __forceinline__ double exp_scaled(const DistillDev& a, double t) { return exp(t * a.inv_tau); }

template <int NT> __device__ __forceinline__ void row_sync() {
    if constexpr (NT == 64) wave_sync(); else __syncthreads();
}

// sums and maxima over the NT threads of a row, in a fixed order; scratch: NT / 64 doubles per value
template <int NT, int Q> __device__ __forceinline__ void row_sum(double (&v)[Q], double* scratch) {
#pragma unroll
    for (int q = 0; q < Q; ++q) v[q] = lanes_reduce<64>(v[q], OpSum());
    if constexpr (NT > 64) {
        constexpr int W = NT / 64;
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
            for (int q = 0; q < Q; ++q) scratch[q * W + wave] = v[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            double s = 0.0;
            for (int i = 0; i < W; ++i) s += scratch[q * W + i];
            v[q] = s;
        }
    }
}
template <int NT, int Q> __device__ __forceinline__ void row_max(double (&v)[Q], double* scratch) {
#pragma unroll
    for (int q = 0; q < Q; ++q) v[q] = lanes_reduce<64>(v[q], OpMax());
    if constexpr (NT > 64) {
        constexpr int W = NT / 64;
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
            for (int q = 0; q < Q; ++q) scratch[q * W + wave] = v[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            double s = scratch[q * W];
            for (int i = 1; i < W; ++i) s = s > scratch[q * W + i] ? s : scratch[q * W + i];
            v[q] = s;
        }
    }
}

// LDS of one row: [bits: V / 32 words][log p: K doubles][student's entries: K doubles][scratch][class: K ints], in 8-byte steps
__host__ __device__ inline size_t distill_lds(int V, int K, int NT) {
    const size_t words = ((size_t)V + 63) / 64 * 2;
    return words * 4 + (size_t)K * 16 + (NT > 64 ? (size_t)NT / 64 * 4 * 8 : 0) + ((size_t)K * 4 + 15) / 16 * 16;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) distill_kernel(DistillDev a) {
    using acc = typename Num<T>::acc;
    constexpr int VN = Vec<T>::N, ROWS = NT < 256 ? 256 / NT : 1;
    extern __shared__ __align__(16) unsigned char lds_all[];
    const int tid = threadIdx.x & (NT - 1);
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT;
    if (row >= a.n) return;                            // ROWS > 1: whole waves, which only wait for themselves
    unsigned char* lds = lds_all + (threadIdx.x / NT) * distill_lds(a.V, a.K, NT);
    const int words = (a.V + 63) / 64 * 2;
    unsigned* bits = reinterpret_cast<unsigned*>(lds);
    double* logp = reinterpret_cast<double*>(lds + (size_t)words * 4);
    double* xtop = logp + a.K;
    double* scratch = xtop + a.K;
    int* cls = reinterpret_cast<int*>(scratch + (NT > 64 ? NT / 64 * 4 : 0));

    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    T* g = a.dlogits ? static_cast<T*>(a.dlogits) + row * a.ld_out : nullptr;
    acc* loss = static_cast<acc*>(a.loss);
    const int nvec = a.V / VN;
    const double w = a.weight ? load_any(a.weight, a.weight_dtype, row) : 1.0;

    auto fill = [&](T value) {
        if (g == nullptr) return;
        typename Vec<T>::raw z;
        for (int i = 0; i < VN; ++i) z[i] = value;
        for (int u = tid; u < nvec; u += NT) Vec<T>::store(g + (size_t)u * VN, z);
        for (int v = nvec * VN + tid; v < a.V; v += NT) g[v] = value;
    };
    if (w == 0.0) { fill((T)0); if (tid == 0) loss[row] = 0; return; }

    // ---- the teacher's entries -------------------------------------------------------------------------------------
    for (int i = tid; i < words; i += NT) bits[i] = 0;
    row_sync<NT>();
    double seen[3] = {0.0, 0.0, 0.0};                  // entries, entries of a class seen before, indices out of range
    for (int k = tid; k < a.K; k += NT) {
        const int64_t c = a.index_64 ? static_cast<const int64_t*>(a.index)[row * a.ld_index + k] : static_cast<const int32_t*>(a.index)[row * a.ld_index + k];
        const double t = load_any(a.top, a.top_dtype, row * a.ld_top + k);
        const bool in = c >= 0 && c < a.V, there = in && !(t == -INFINITY);
        if (there) {
            const unsigned before = atomicOr(&bits[c >> 5], 1u << (c & 31));
            seen[0] += 1.0;
            seen[1] += before >> (c & 31) & 1 ? 1.0 : 0.0;
            logp[k] = t * a.inv_tau;
            xtop[k] = (double)(acc)x[c];
        }
        if (!in && c != -1) seen[2] += 1.0;
        cls[k] = there ? (int)c : -1;
    }
    row_sum<NT>(seen, scratch);
    if (seen[2] > 0.0) { fill((T)NAN); if (tid == 0) loss[row] = NAN; return; }
    if (seen[0] == 0.0) { fill((T)0); if (tid == 0) loss[row] = 0; return; }
    row_sync<NT>();
    if (seen[1] > 0.0) {
        // entries of one class: the first takes the logarithm of their sum, the others become padding
        constexpr int PER = (OAK_MAX_TEACHER + NT - 1) / NT;
        double merged[PER]; int keep = 0;
        int q = 0;
        for (int k = tid; k < a.K; k += NT, ++q) {
            const int c = cls[k];
            bool first = c >= 0;
            double m = -INFINITY, s = 0.0;
            for (int i = 0; c >= 0 && i < a.K; ++i) {
                if (cls[i] != c) continue;
                if (i < k) first = false;
                m = logp[i] > m ? logp[i] : m;
            }
            for (int i = 0; first && i < a.K; ++i) if (cls[i] == c) s += exp(logp[i] - m);
            if (q < PER) merged[q] = m + log(s);
            keep |= first ? 1 << q : 0;
        }
        row_sync<NT>();
        q = 0;
        for (int k = tid; k < a.K; k += NT, ++q) {
            if (keep >> q & 1) logp[k] = merged[q]; else cls[k] = -1;
        }
        row_sync<NT>();
    }
    const bool some_rest = seen[0] - seen[1] < (double)a.V;
    double zt = 0.0;
    if (a.lse) zt = load_any(a.lse, a.lse_dtype, row);
    else {
        double m[1] = {-INFINITY}, s[1] = {0.0};
        for (int k = tid; k < a.K; k += NT) if (cls[k] >= 0) m[0] = logp[k] > m[0] ? logp[k] : m[0];
        row_max<NT>(m, scratch);
        for (int k = tid; k < a.K; k += NT) if (cls[k] >= 0) s[0] += exp(logp[k] - m[0]);
        row_sum<NT>(s, scratch);
        zt = m[0] + log(s[0]);
    }

    // ---- one pass over the classes: maximum and sum of the rest ------------------------------------------------------
    constexpr acc LOWEST = sizeof(acc) == 8 ? (acc)-1.7976931348623157e308 : (acc)-3.402823466e38f;
    acc m = LOWEST, z = 0;                             // a finite start: -inf - m stays -inf
    auto take = [&](const acc (&v)[VN]) {
        acc top = m;
#pragma unroll
        for (int i = 0; i < VN; ++i) top = v[i] > top ? v[i] : top;
        z *= exp_scaled(a, m - top);
        m = top;
#pragma unroll
        for (int i = 0; i < VN; ++i) z += exp_scaled(a, v[i] - m);
    };
    auto bits_of = [&](int u) {                         // the VN bits of unit u
        const int v = u * VN;
        return bits[v >> 5] >> (v & 31);
    };
    for (int u = tid; u < nvec; u += NT) {
        const auto r = Vec<T>::load(x + (size_t)u * VN);
        const unsigned b = bits_of(u);
        acc v[VN];
#pragma unroll
        for (int i = 0; i < VN; ++i) v[i] = b >> i & 1 ? (acc)-INFINITY : (acc)r[i];
        take(v);
    }
    {
        acc v[VN];
        const int at = nvec * VN + tid;
#pragma unroll
        for (int i = 0; i < VN; ++i) v[i] = -INFINITY;
        if (at < a.V && tid < VN && !(bits[at >> 5] >> (at & 31) & 1)) v[0] = (acc)x[at];
        if (tid < VN) take(v);
    }

    // ---- the row's numbers -----------------------------------------------------------------------------------------
    double top2[2] = {(double)m, -INFINITY};
    for (int k = tid; k < a.K; k += NT) if (cls[k] >= 0) top2[1] = xtop[k] > top2[1] ? xtop[k] : top2[1];
    row_max<NT>(top2, scratch);
    const double mr = top2[0], M = mr > top2[1] ? mr : top2[1];
    double s3[3] = {(double)z * exp(((double)m - mr) * a.inv_tau), 0.0, 0.0};     // rest (on mr), top (on M), sum p
    for (int k = tid; k < a.K; k += NT) if (cls[k] >= 0) {
        s3[1] += exp((xtop[k] - M) * a.inv_tau);
        s3[2] += exp(logp[k] - zt);
    }
    row_sum<NT>(s3, scratch);
    const double logz = log(s3[0] * exp((mr - M) * a.inv_tau) + s3[1]);           // on M
    const bool rest = a.lse != nullptr && some_rest;
    double pr = 0.0;
    const double lqr = (mr - M) * a.inv_tau + log(s3[0]) - logz, qr = some_rest ? exp(lqr) : 0.0;
    if (rest) {
        pr = 1.0 - s3[2];
        pr = pr < 0.0 ? 0.0 : pr;
    }
    double kl[1] = {0.0};
    for (int k = tid; k < a.K; k += NT) if (cls[k] >= 0) {
        const double lp = logp[k] - zt, lq = (xtop[k] - M) * a.inv_tau - logz;
        const double weight = exp(a.reverse ? lq : lp);
        if (weight != 0.0) kl[0] += a.reverse ? weight * (lq - lp) : weight * (lp - lq);
    }
    row_sum<NT>(kl, scratch);
    // the rest's gradient is mass_r e_v / sum e over the rest, e_v = exp((s_v - m_r) / tau): q_v (1 - p_r / q_r) would be 0 times infinity
    // where the student is sure of itself
    double mass_r = qr;
    if (a.reverse) {
        const double lr = rest ? lqr - log(pr > a.floor_rest ? pr : a.floor_rest) : 0.0;
        if (qr != 0.0) kl[0] += qr * lr;
        mass_r = qr * (lr - kl[0]);
    } else if (rest && pr > 0.0) {
        kl[0] += pr * (log(pr) - lqr);
        mass_r = qr - pr;
    }
    if (tid == 0) loss[row] = (acc)(a.tau * a.tau * w * kl[0]);
    if (g == nullptr) return;

    // ---- the gradient: the rest's coefficient everywhere, then the entries' own values over it ------------------------
    const acc coef = (acc)(s3[0] == 0.0 ? 0.0 : a.tau * w * mass_r / s3[0]), mm = (acc)mr;
    for (int u = tid; u < nvec; u += NT) {
        const auto r = Vec<T>::load(x + (size_t)u * VN);
        typename Vec<T>::raw o;
#pragma unroll
        for (int i = 0; i < VN; ++i) o[i] = (T)(coef * exp_scaled(a, (acc)r[i] - mm));
        Vec<T>::store(g + (size_t)u * VN, o);
    }
    if (nvec * VN + tid < a.V && tid < VN) g[nvec * VN + tid] = (T)(coef * exp_scaled(a, (acc)x[nvec * VN + tid] - mm));
    row_sync<NT>();
    for (int k = tid; k < a.K; k += NT) if (cls[k] >= 0) {
        const double lp = logp[k] - zt, lq = (xtop[k] - M) * a.inv_tau - logz, q = exp(lq);
        const double d = a.reverse ? (q != 0.0 ? q * (lq - lp - kl[0]) : 0.0) : q - exp(lp);
        g[cls[k]] = (T)(acc)(a.tau * w * d);
    }
}

static int distill_check(const oak_distill_args* a) {
    OAK_REQUIRE(a != nullptr, "distill: arguments are NULL");
    OAK_REQUIRE(a->n_rows >= 0 && a->n_rows < ((int64_t)1 << 31), "distill: n_rows = %lld", (long long)a->n_rows);
    OAK_REQUIRE(a->n_classes >= 1 && a->n_classes <= OAK_MAX_CLASSES, "distill: n_classes = %d is not in 1 .. %d", a->n_classes, OAK_MAX_CLASSES);
    OAK_REQUIRE(a->top_k >= 1 && a->top_k <= OAK_MAX_TEACHER, "distill: top_k = %d is not in 1 .. %d", a->top_k, OAK_MAX_TEACHER);
    OAK_REQUIRE(a->dtype >= OAK_F64 && a->dtype <= OAK_F16 && a->top_dtype >= OAK_F64 && a->top_dtype <= OAK_F16, "distill: unknown element type");
    OAK_REQUIRE((!a->top_lse || (a->lse_dtype >= OAK_F64 && a->lse_dtype <= OAK_F16)) &&
                (!a->row_weight || (a->weight_dtype >= OAK_F64 && a->weight_dtype <= OAK_F16)), "distill: unknown element type");
    OAK_REQUIRE(a->direction == OAK_KL_FORWARD || a->direction == OAK_KL_REVERSE, "distill: unknown direction %d", a->direction);
    OAK_REQUIRE(a->direction == OAK_KL_FORWARD || a->top_lse, "distill: the reverse direction needs top_lse");
    OAK_REQUIRE(a->temperature > 0.0 && a->temperature - a->temperature == 0.0, "distill: temperature must be positive and finite");
    OAK_REQUIRE(a->temperature >= 1e-6 && a->temperature <= 1e6, "distill: temperature %g is not in 1e-6 .. 1e6", a->temperature);
    OAK_REQUIRE(a->n_rows == 0 || (a->logits && a->top && a->index && a->loss), "distill: an array is NULL");
    OAK_REQUIRE(a->n_rows <= 1 || (a->ld_logits >= 0 && a->ld_top >= 0 && a->ld_index >= 0), "distill: negative row stride");
    OAK_REQUIRE(a->n_rows <= 1 || !a->dlogits || a->ld_dlogits >= a->n_classes, "distill: rows of dlogits overlap");
    return OAK_OK;
}

template <typename T, int NT> static int distill_run(hipStream_t stream, const DistillDev& d) {
    constexpr int ROWS = NT < 256 ? 256 / NT : 1;
    const size_t lds = (distill_lds(d.V, d.K, NT)) * ROWS;
    auto kernel = distill_kernel<T, NT>;
    if (lds > 64 * 1024) OAK_CHECK(ensure_dynamic_lds((const void*)kernel, 160 * 1024));
    return launch(kernel, dim3((unsigned)((d.n + ROWS - 1) / ROWS)), dim3(NT < 256 ? 256 : NT), lds, stream, d);
}

static int distill_launch(hipStream_t stream, const oak_distill_args* a) {
    if (a->n_rows == 0) return OAK_OK;
    DistillDev d{};
    d.n = a->n_rows; d.ld = a->ld_logits; d.ld_top = a->ld_top; d.ld_index = a->ld_index; d.ld_out = a->ld_dlogits;
    d.V = a->n_classes; d.K = a->top_k; d.top_dtype = a->top_dtype; d.lse_dtype = a->lse_dtype; d.weight_dtype = a->weight_dtype;
    d.index_64 = a->index_64; d.reverse = a->direction == OAK_KL_REVERSE;
    d.tau = a->temperature; d.inv_tau = 1.0 / a->temperature; d.floor_rest = a->dtype == OAK_F64 ? 0x1p-53 : 0x1p-24;
    const double c = 1.4426950408889634074 / a->temperature;
    d.c_hi = (float)c;
    if ((double)d.c_hi >= c) d.c_hi = __builtin_nextafterf(d.c_hi, 0.0f);
    d.c_lo = (float)(c - (double)d.c_hi);
    d.logits = a->logits; d.top = a->top; d.index = a->index; d.lse = a->top_lse; d.weight = a->row_weight; d.loss = a->loss; d.dlogits = a->dlogits;
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        if (d.V <= 1024 && d.K <= 256) return distill_run<T, 64>(stream, d);
        return distill_run<T, 256>(stream, d);
    });
}

}  // namespace oak

using namespace oak;

extern "C" {

int oak_device_pointer_check(int32_t device, const void* p) {
    return c_entry([&] {
        OAK_REQUIRE(p != nullptr, "the pointer is NULL");
        hipPointerAttribute_t at{};
        const hipError_t e = hipPointerGetAttributes(&at, p);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            OAK_REQUIRE(false, "%p is not memory of this library's HIP runtime (%s)", p, hipGetErrorString(e));
        }
        OAK_REQUIRE((at.type == hipMemoryTypeDevice || at.type == hipMemoryTypeManaged) && at.device == device,
                    "%p is not memory of device %d known to this library's HIP runtime", p, device);
        return (int)OAK_OK;
    });
}

int oak_distill_device(int32_t device, void* stream, const oak_distill_args* a) {
    return c_entry([&] {
        OAK_CHECK(distill_check(a));
        DeviceGuard g;
        OAK_CHECK(g.enter(device));
        return distill_launch((hipStream_t)stream, a);
    });
}

int oak_distill(oak_ctx* ctx, const oak_distill_args* args) {
    return c_entry([&] {
        if (!ctx) { set_error("ctx is NULL"); return OAK_E_ARG; }
        OAK_CHECK(distill_check(args));
        OAK_REQUIRE(args->dtype == OAK_F64 && args->top_dtype == OAK_F64 && (!args->top_lse || args->lse_dtype == OAK_F64) &&
                    (!args->row_weight || args->weight_dtype == OAK_F64) && args->ld_logits == args->n_classes && args->ld_top == args->top_k &&
                    args->ld_index == args->top_k && (!args->dlogits || args->ld_dlogits == args->n_classes),
                    "distill: host arrays are contiguous float64");
        OAK_HIP_CHECK(hipSetDevice(ctx->device));
        if (args->n_rows == 0) return (int)OAK_OK;
        PhaseTimer t(ctx, "distill");
        oak_distill_args a = *args;
        HostStage st(ctx);
        const size_t n = (size_t)a.n_rows, cells = n * a.n_classes, kept = n * a.top_k;
        OAK_CHECK(st.in("kd_logits", a.logits, cells * 8));
        OAK_CHECK(st.in("kd_top", a.top, kept * 8));
        OAK_CHECK(st.in("kd_index", a.index, kept * (a.index_64 ? 8 : 4)));
        OAK_CHECK(st.in("kd_lse", a.top_lse, n * 8));
        OAK_CHECK(st.in("kd_weight", a.row_weight, n * 8));
        OAK_CHECK(st.out("kd_loss", a.loss, n * 8));
        OAK_CHECK(st.out("kd_dlogits", a.dlogits, cells * 8));
        OAK_CHECK(distill_launch(ctx->stream, &a));
        t.stop();
        return st.finish();
    });
}

}  // extern "C"
