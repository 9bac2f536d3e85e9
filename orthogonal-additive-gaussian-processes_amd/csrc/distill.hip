// Divergence of a student's class distribution from a teacher's top logits, and its gradient.
//
// With z = log sum_v exp(s_v / tau), q_v = exp(s_v / tau - z), "top" the teacher's entries and "rest" every other class:
//   forward  L = tau^2 w [ sum p_k (log p_k - log q_k) + p_r (log p_r - log q_r) ]
//            dL/ds_v = tau w (S q_v - p_v) on the top,  tau w q_v (S - p_r / q_r) on the rest   (p_r = 0 without a rest outcome; S = sum p_k + p_r,
//            1 unless the entries' own sum passes 1, as with a top_lse of 16 bits, or they are all the classes.  Off by less than 2^-18, as single
//            precision leaves a top_lse of up to 32, it is taken for the 1 that it stands for)
//   reverse  L = tau^2 w [ sum q_k (log q_k - log p_k) + q_r (log q_r - log p_r) ]
//            dL/ds_v = tau w q_v (log q_b - log p_b - L / (tau^2 w)),  b the outcome v belongs to
// so the gradient is one coefficient times q_v on the rest and k values of their own on the top.
//
// q_r is summed over the rest itself (the teacher's entries left out, found by a bit per class in LDS): taken as 1 - sum q_k it would lose
// every digit where the student is sure of itself, and so would log z next to one sure class.  Exponentials and the sum over the 4 or 8 classes
// of a 16-byte unit are 32 bits (64 for double), everything across units, per entry and per row is 64: a lane takes up to 2048 classes, and a flat
// row rounds alike at every step of a running sum in 32 bits (1e-5 of the sum at 2^20 classes).
//
// A row stays in the registers of its team of NT threads, NV units of 16 bytes each, so that it is read once: the sum and the gradient
// each walk the registers (LONG: what does not fit is read twice).  The team's first wave (all of a smaller team) does what concerns the entries.
// Every sum over the entries is taken on
// references known before the pass over the classes (the entries' own maximum), so that only one reduction per row waits for that pass.
#include "lowp.h"

namespace oak {

struct DistillDev {
    int64_t n, ld, ld_top, ld_index, ld_out;
    int V, K, top_dtype, lse_dtype, weight_dtype, index_64, reverse;
    double tau, inv_tau, floor_rest;
    float c_hi, c_lo;           // log2(e) / tau in two floats, c_hi rounded towards zero
    const void* logits; const void* top; const void* index; const void* lse; const void* weight;
    void* loss; void* dlogits;
    double* part;               // split rows: maximum and sum of every slice [n][slices][2]
    int slices, slice;          // and the units of a slice
};

// exp(t / tau) for t <= 0.  float: 2^(t c) with c in two parts, since a c off by half a unit would put a common relative error of |t| c 2^-25
// on all the terms of a sum (t = 20: 1e-6 in log z, more than a small divergence bears).  Both parts are positive: t = -inf gives 0, NaN stays NaN.
__device__ __forceinline__ float exp_scaled(const DistillDev& a, float t) { return __builtin_amdgcn_exp2f(__builtin_fmaf(t, a.c_hi, t * a.c_lo)); }
__device__ __forceinline__ double exp_scaled(const DistillDev& a, double t) { return exp_of(t * a.inv_tau); }
// for a gradient of type T: one part of c is enough for 16 bits
template <typename T> __device__ __forceinline__ typename Num<T>::acc exp_gradient(const DistillDev& a, typename Num<T>::acc t) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(t * a.c_hi); else return exp_scaled(a, t);
}

// LDS of one team, in 8-byte steps: [bits: one a class][t - reference][p][exp((x - x_ref) / tau)][waves' maxima and sums, row's numbers][class]
__host__ __device__ inline size_t distill_words(int V) { return ((size_t)V + 63) / 64 * 2; }
__host__ __device__ inline size_t distill_lds(int V, int K, int NT) {
    return distill_words(V) * 4 + (size_t)K * 24 + (NT > 64 ? (size_t)(NT / 64 * 2 + 4) * 8 : 0) + ((size_t)K * 4 + 15) / 16 * 16;
}

// what the team does with its row's gradient
enum { ROW_COMPUTE = 0, ROW_ZERO = 1, ROW_NAN = 2 };

// where a team's row is: in its registers; there and, what does not fit, read twice; cut into slices, a workgroup each, whose sums
// distill_slice_kernel has made
enum { HELD = 0, LONG = 1, SPLIT = 2 };

__device__ __forceinline__ float lowest(float) { return -3.402823466e38f; }
__device__ __forceinline__ double lowest(double) { return -1.7976931348623157e308; }

// a unit with the elements of the bits set in b replaced by -inf; two 16-bit elements at a time
template <typename T> __device__ __forceinline__ typename Vec<T>::raw hidden(typename Vec<T>::raw r, unsigned b) {
    if constexpr (sizeof(T) == 2) {
        typedef unsigned words4 __attribute__((ext_vector_type(4)));
        words4 w = __builtin_bit_cast(words4, r);
        const unsigned inf = (unsigned)__builtin_bit_cast(unsigned short, (T)-INFINITY) * 0x10001u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned low = (unsigned)((int)(b << (31 - 2 * i)) >> 31), high = (unsigned)((int)(b << (30 - 2 * i)) >> 31);
            const unsigned mask = (low & 0xffffu) | (high & 0xffff0000u);
            w[i] = (inf & mask) | (w[i] & ~mask);
        }
        return __builtin_bit_cast(typename Vec<T>::raw, w);
    } else {
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i) r[i] = b >> i & 1 ? (T)-INFINITY : r[i];
        return r;
    }
}

// sum over one unit, on m
template <int VN, typename A, typename R> __device__ __forceinline__ A sum_unit(const DistillDev& a, const R& r, A m) {
    A sum = exp_scaled(a, (A)r[0] - m);
#pragma unroll
    for (int j = 1; j < VN; ++j) sum += exp_scaled(a, (A)r[j] - m);
    return sum;
}
// one more unit into a running maximum m and sum z
template <int VN, typename A, typename R> __device__ __forceinline__ void take_unit(const DistillDev& a, const R& r, A& m, double& z) {
    A top = m;
#pragma unroll
    for (int j = 0; j < VN; ++j) top = OpMax()(top, (A)r[j]);
    z = z * (double)exp_scaled(a, m - top) + (double)sum_unit<VN>(a, r, top);
    m = top;
}

// Few rows: maximum and sum of the rest over one slice of one row.
template <typename T, int NT> __global__ void __launch_bounds__(NT) distill_slice_kernel(DistillDev a) {
    using acc = typename Num<T>::acc;
    constexpr int VN = Vec<T>::N, U = 4;
    extern __shared__ __align__(16) unsigned char lds_all[];
    __shared__ double share[NT / 64][2];
    unsigned* bits = reinterpret_cast<unsigned*>(lds_all);
    const int tid = threadIdx.x, nvec = a.V / VN, u_begin = blockIdx.x * a.slice, u_end = u_begin + a.slice < nvec ? u_begin + a.slice : nvec;
    const bool last_slice = blockIdx.x + 1 == gridDim.x;
    const int64_t row = blockIdx.y;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    if (a.weight && load_any(a.weight, a.weight_dtype, row) == 0.0) return;
    const int64_t v_begin = (int64_t)u_begin * VN, v_end = last_slice ? a.V : (int64_t)u_end * VN;
    for (int i = tid; i < (int)((v_end - v_begin + 31) / 32); i += NT) bits[i] = 0;
    __syncthreads();
    for (int k = tid; k < a.K; k += NT) {
        const int64_t c = a.index_64 ? static_cast<const int64_t*>(a.index)[row * a.ld_index + k] : static_cast<const int32_t*>(a.index)[row * a.ld_index + k];
        if (c >= v_begin && c < v_end && !(load_any(a.top, a.top_dtype, row * a.ld_top + k) == -INFINITY))
            atomicOr(&bits[(c - v_begin) >> 5], 1u << ((c - v_begin) & 31));
    }
    __syncthreads();
    acc m = lowest(acc());
    double z = 0.0;
    for (int u0 = u_begin + tid; u0 < u_end; u0 += U * NT) {
        typename Vec<T>::raw r[U];
#pragma unroll
        for (int i = 0; i < U; ++i) { const int u = u0 + i * NT; r[i] = Vec<T>::load(x + (size_t)(u < u_end ? u : u_end - 1) * VN); }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = u0 + i * NT;
            if (u >= u_end) break;
            const int v = (u - u_begin) * VN;
            const unsigned b = bits[v >> 5] >> (v & 31);
            r[i] = hidden<T>(r[i], b);
            take_unit<VN>(a, r[i], m, z);
        }
    }
    const int64_t extra = (int64_t)nvec * VN + tid;                                // elements that do not fill a unit
    if (last_slice && extra < a.V && !(bits[(extra - v_begin) >> 5] >> ((extra - v_begin) & 31) & 1)) {
        const acc one[1] = {(acc)x[extra]};
        take_unit<1>(a, one, m, z);
    }
    const acc mw = lanes_reduce<64>(m, OpMax());
    const double zw = lanes_reduce<64>(z * (double)exp_scaled(a, m - mw), OpSum());
    if ((tid & 63) == 0) { share[tid >> 6][0] = (double)mw; share[tid >> 6][1] = zw; }
    __syncthreads();
    if (tid < NT / 64) {
        const double mine = share[tid][0], all = lanes_reduce<NT / 64>(mine, OpMax());
        const double sum = lanes_reduce<NT / 64>(share[tid][1] * exp_of((mine - all) * a.inv_tau), OpSum());
        if (tid == 0) { double* p = a.part + (row * a.slices + blockIdx.x) * 2; p[0] = all; p[1] = sum; }
    }
}

template <typename T, int NT, int NV, int MODE>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT, MODE == LONG ? 4 : 1) distill_kernel(DistillDev a) {
    using acc = typename Num<T>::acc;
    using raw = typename Vec<T>::raw;
    constexpr int VN = Vec<T>::N, ROWS = NT < 256 ? 256 / NT : 1, LEAD = NT < 64 ? NT : 64, WAVES = NT / 64;
    static_assert(NT >= VN, "a thread for every element that does not fill a unit");
    extern __shared__ __align__(16) unsigned char lds_all[];
    const int tid = threadIdx.x & (NT - 1);
    unsigned char* lds = lds_all + (NT < 256 ? threadIdx.x / NT : 0) * distill_lds(a.V, a.K, NT);
    const int words = (int)distill_words(a.V);
    unsigned* bits = reinterpret_cast<unsigned*>(lds);
    double* tk = reinterpret_cast<double*>(lds + (size_t)words * 4);
    double* pk = tk + a.K;
    double* ek = pk + a.K;
    double* share = ek + a.K;
    int* cls = reinterpret_cast<int*>(share + (NT > 64 ? WAVES * 2 + 4 : 0));
    const int nvec = a.V / VN;
    // the units read from memory (not held), and the elements that do not fill one
    const int u_begin = MODE == SPLIT ? blockIdx.x * a.slice : NV * NT, u_end = MODE == SPLIT && u_begin + a.slice < nvec ? u_begin + a.slice : nvec;
    const int tail = MODE == SPLIT && blockIdx.x + 1 != gridDim.x ? 0 : a.V - nvec * VN;
    const bool lead = tid < LEAD;
    auto team_sync = [] { if constexpr (NT <= 64) wave_sync(); else __syncthreads(); };

    for (int i = tid; i < words; i += NT) bits[i] = 0;
    team_sync();

    const int64_t stride = MODE == SPLIT ? a.n : (int64_t)gridDim.x * ROWS;
    for (int64_t row = MODE == SPLIT ? (int64_t)blockIdx.y : (int64_t)blockIdx.x * ROWS + (NT < 256 ? threadIdx.x / NT : 0); row < a.n; row += stride) {
        const T* x = static_cast<const T*>(a.logits) + row * a.ld;
        T* g = a.dlogits ? static_cast<T*>(a.dlogits) + row * a.ld_out : nullptr;
        const double w = a.weight ? load_any(a.weight, a.weight_dtype, row) : 1.0;
        int todo = w == 0.0 ? ROW_ZERO : ROW_COMPUTE;

        // this lane's place, forgotten by the compiler now and then: it would otherwise keep the NV addresses, offsets and bit positions of a
        // lane in registers from row to row
        int at = tid;
        auto forget_place = [&] { asm volatile("" : "+v"(at)); };
        forget_place();
        // ---- the row into registers; units behind its end are read from inside it and not used -----------------------------
        typedef int words4 __attribute__((ext_vector_type(4)));
        words4 data[NV];
        acc last = -INFINITY;                          // one of the elements that do not fill a unit
        if (todo == ROW_COMPUTE) {
            if (MODE != SPLIT && nvec > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int u = i * NT + at;
                    data[i] = __builtin_bit_cast(words4, Vec<T>::load(x + (size_t)(u < nvec ? u : nvec - 1) * VN));
                }
            }
            if (tid < tail) last = (acc)x[nvec * VN + tid];
        }

        // ---- the teacher's entries ------------------------------------------------------------------------------------
        double xref = -INFINITY, ref = 0.0, sums[6] = {0, 0, 0, 0, 0, 0};        // sum e, e (t - ref), e (x - xref); f, f (x - xref), f (t - ref)
        bool some_rest = true;
        if (lead && todo == ROW_COMPUTE) {
            unsigned count = 0, again = 0, wrong = 0;
            double tmax = -INFINITY;
            for (int k = tid; k < a.K; k += LEAD) {
                const int64_t c = a.index_64 ? static_cast<const int64_t*>(a.index)[row * a.ld_index + k] : static_cast<const int32_t*>(a.index)[row * a.ld_index + k];
                const double kept = load_any(a.top, a.top_dtype, row * a.ld_top + k), scaled = kept * a.inv_tau;
                const double t = scaled < lowest(double()) ? lowest(double()) : scaled;      // a value that is not -inf is an entry at any temperature
                const bool in = c >= 0 && c < a.V, there = in && !(kept == -INFINITY);
                wrong |= !in && c != -1 ? 1u : 0u;
                cls[k] = there ? (int)c : -1;
                if (there) {
                    const unsigned before = atomicOr(&bits[c >> 5], 1u << (c & 31));
                    ++count;
                    again += before >> (c & 31) & 1;
                    const double xe = (double)(acc)x[c];
                    tk[k] = t; ek[k] = xe;
                    tmax = __builtin_fmax(tmax, t); xref = __builtin_fmax(xref, xe);
                }
            }
            count = lanes_reduce<LEAD>(count, OpSum());
            again = lanes_reduce<LEAD>(again, OpSum());
            wrong = lanes_reduce<LEAD>(wrong, OpOr());
            some_rest = count - again < (unsigned)a.V;
            todo = wrong ? ROW_NAN : count == 0 ? ROW_ZERO : ROW_COMPUTE;
            wave_sync();
            if (again > 0) {
                // entries of one class: the first takes the logarithm of their sum, the others become padding
                for (int k = tid; k < a.K; k += LEAD) {
                    const int c = cls[k];
                    bool first = c >= 0;
                    double m = -INFINITY, s = 0.0;
                    for (int i = 0; c >= 0 && i < a.K; ++i) {
                        if (cls[i] != c) continue;
                        if (i < k) first = false;
                        m = __builtin_fmax(m, tk[i]);
                    }
                    for (int i = 0; first && i < a.K; ++i) if (cls[i] == c) s += exp_of(tk[i] - m);
                    pk[k] = first ? m + log_of(s) : -INFINITY;
                }
                wave_sync();
                for (int k = tid; k < a.K; k += LEAD) {
                    if (pk[k] == -INFINITY) cls[k] = -1; else { tk[k] = pk[k]; tmax = __builtin_fmax(tmax, pk[k]); }
                }
            }
            ref = a.lse ? load_any(a.lse, a.lse_dtype, row) : lanes_reduce<LEAD>(tmax, OpMax());
            xref = __builtin_fmax(lanes_reduce<LEAD>(xref, OpMax()), -1e300);
            for (int k = tid; k < a.K; k += LEAD) if (cls[k] >= 0) {
                const double dt = tk[k] - ref, dx = ek[k] - xref, e = exp_of(dt > 1000.0 ? 1000.0 : dt), f = exp_of(dx * a.inv_tau);   // a top_lse far below its entries: no finite loss
                tk[k] = dt; pk[k] = e; ek[k] = f;
                sums[0] += e;
                if (e != 0.0) { sums[1] += e * dt; sums[2] += e * dx; }
                sums[3] += f;
                if (f != 0.0 && a.reverse) { sums[4] += f * dx; sums[5] += f * dt; }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) sums[q] = lanes_reduce<LEAD>(sums[q], OpSum());
            if (a.reverse) { sums[4] = lanes_reduce<LEAD>(sums[4], OpSum()); sums[5] = lanes_reduce<LEAD>(sums[5], OpSum()); }
        }
        if constexpr (NT > 64) {
            if (tid == 0) share[WAVES * 2] = (double)todo;
            __syncthreads();
            todo = (int)share[WAVES * 2];
        }

        acc m = lowest(acc());                         // a finite start: -inf - m stays -inf
        double z = 0.0;
        if (MODE != SPLIT && todo == ROW_COMPUTE) {
            auto forget = [&] {                         // the units, not their 32-bit forms, live from one walk to the next
#pragma unroll
                for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(data[i]));
                forget_place();
            };
            // ---- maximum and sum of the rest -----------------------------------------------------------------------------------
            auto hide = [&](raw& r, int u) {            // the entries' classes become -inf; their gradients are written over at the end
                const int v = u * VN;
                const unsigned b = bits[v >> 5] >> (v & 31) & ((1u << VN) - 1);
                if (__any(b != 0)) r = hidden<T>(r, b);
            };
            if (tid < tail && (bits[(nvec * VN + tid) >> 5] >> ((nvec * VN + tid) & 31) & 1)) last = -INFINITY;
            {
                forget_place();
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int u = i * NT + at;
                    if (u < nvec) {
                        raw r = __builtin_bit_cast(raw, data[i]);
                        hide(r, u);
                        data[i] = __builtin_bit_cast(words4, r);
#pragma unroll
                        for (int j = 0; j < VN; ++j) m = OpMax()(m, (acc)r[j]);
                    }
                    __builtin_amdgcn_sched_barrier(0);      // one unit at a time: the registers hold the row
                }
                m = OpMax()(m, last);
                forget();
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (i * NT + at < nvec) {
                        z += (double)sum_unit<VN>(a, __builtin_bit_cast(raw, data[i]), m);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                z += (double)exp_scaled(a, last - m);
                forget();
            }
            if constexpr (MODE == LONG) {
                constexpr int U = 4;
                for (int u0 = u_begin + tid; u0 < nvec; u0 += U * NT) {
                    raw r[U];
#pragma unroll
                    for (int i = 0; i < U; ++i) { const int u = u0 + i * NT; r[i] = Vec<T>::load(x + (size_t)(u < nvec ? u : nvec - 1) * VN); }
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        const int u = u0 + i * NT;
                        if (u < nvec) { hide(r[i], u); take_unit<VN>(a, r[i], m, z); }
                    }
                }
            }
        }
        // ---- across the team -------------------------------------------------------------------------------------------
        acc mr = lanes_reduce<LEAD>(m, OpMax());
        double zr = lanes_reduce<LEAD>(z * (double)exp_scaled(a, m - mr), OpSum());
        if constexpr (MODE == SPLIT) {
            if (lead && todo == ROW_COMPUTE) {
                const double* p = a.part + row * a.slices * 2;
                const double mw = tid < a.slices ? p[tid * 2] : (double)lowest(acc()), all = lanes_reduce<64>(mw, OpMax());
                zr = lanes_reduce<64>(tid < a.slices ? p[tid * 2 + 1] * exp_of((mw - all) * a.inv_tau) : 0.0, OpSum());
                mr = (acc)all;
            }
        } else if constexpr (NT > 64) {
            if ((tid & 63) == 0) { share[tid >> 6] = (double)mr; share[WAVES + (tid >> 6)] = zr; }
            __syncthreads();
            if (lead) {
                // every block of WAVES lanes reduces the same numbers: all lanes have the result
                const double mw = share[tid & (WAVES - 1)], all = lanes_reduce<WAVES>(mw, OpMax());
                zr = lanes_reduce<WAVES>(share[WAVES + (tid & (WAVES - 1))] * exp_of((mw - all) * a.inv_tau), OpSum());
                mr = (acc)all;
            }
        }

        // ---- the row's numbers -----------------------------------------------------------------------------------------
        double log_z = 0.0, kl = 0.0, coef = 0.0, psum = 1.0, total = 1.0;        // log_z on xref, total the teacher's mass
        if (lead && todo == ROW_COMPUTE) {
            const double far = ((double)mr - xref) * a.inv_tau, log_zr = log_of(zr);
            const bool rest = a.lse != nullptr && some_rest;
            // z over all classes: the rest of 32-bit exponentials, the entries of 64-bit ones.  Next to a sure student's entry (z = 1 + little) the little keeps its digits
            log_z = far > 0.0 ? far + log_of(zr + sums[3] * exp_of(-far)) : log_of(zr * exp_of(far) + sums[3]);
            const double lqr = far + log_zr - log_z, qr = some_rest ? exp_of(lqr) : 0.0;
            double pr = 0.0, mass;
            if (a.lse == nullptr) {
                psum = sums[0];
                kl = (sums[1] - sums[2] * a.inv_tau) / psum - log_of(psum) + log_z;
            } else {
                pr = rest ? 1.0 - sums[0] : 0.0;
                pr = pr < 0.0 ? 0.0 : pr;
                total = pr > 0.0 || __builtin_fabs(sums[0] - 1.0) < 0x1p-18 ? 1.0 : sums[0];
                kl = sums[1] - sums[2] * a.inv_tau + sums[0] * log_z;
            }
            if (a.reverse) {
                const double scale = exp_of(-log_z), lr = rest ? lqr - log_of(pr > a.floor_rest ? pr : a.floor_rest) : 0.0;
                kl = scale != 0.0 ? scale * (sums[4] * a.inv_tau - sums[5] - sums[3] * log_z) : 0.0;
                if (qr != 0.0) kl += qr * lr;
                mass = qr != 0.0 ? qr * (lr - kl) : 0.0;
            } else {
                if (pr > 0.0) kl += pr * (log_of(pr) - lqr);
                mass = total * qr - pr;
            }
            // mass e_v / sum e on the rest, e_v = exp((s_v - m_r) / tau): q_v (S - p_r / q_r) would be 0 times infinity where the student is
            // sure of itself
            coef = zr == 0.0 ? 0.0 : mass / zr;
            coef *= a.tau * w;
        }
        if (tid == 0 && (MODE != SPLIT || blockIdx.x == 0)) static_cast<acc*>(a.loss)[row] = todo == ROW_COMPUTE ? (acc)(a.tau * a.tau * w * kl) : todo == ROW_ZERO ? (acc)0 : (acc)NAN;
        if (g != nullptr) {
            if constexpr (NT > 64) {
                if (tid == 0) { share[WAVES * 2 + 1] = coef; share[WAVES * 2 + 2] = (double)mr; }
                __syncthreads();
                coef = share[WAVES * 2 + 1]; mr = (acc)share[WAVES * 2 + 2];
            }
            // ---- the gradient: the rest's coefficient everywhere, then the entries' own values over it ------------------------
            const acc cf = (acc)coef, fill = todo == ROW_NAN ? (acc)NAN : (acc)0;
            auto put = [&](const raw& r, int u) {
                raw o;
#pragma unroll
                for (int j = 0; j < VN; ++j) o[j] = (T)(todo == ROW_COMPUTE ? cf * exp_gradient<T>(a, (acc)r[j] - mr) : fill);
                // a long row's gradient passes the caches by (16384 x 8192 bf16: 140 us, otherwise 158); short rows end inside a cache line, which
                // the next row fills there (262144 x 1000 float32: 430 us, otherwise 510)
                if constexpr (MODE != HELD || NT * NV >= 1024) Vec<T>::store_stream(g + (size_t)u * VN, o); else Vec<T>::store(g + (size_t)u * VN, o);
            };
            if constexpr (MODE != SPLIT) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int u = i * NT + at;
                    if (u < nvec) put(__builtin_bit_cast(raw, data[i]), u);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (MODE != HELD) {
                constexpr int U = 4;
                for (int u0 = u_begin + tid; u0 < u_end; u0 += U * NT) {
                    raw r[U] = {};
                    if (todo == ROW_COMPUTE) {
#pragma unroll
                        for (int i = 0; i < U; ++i) { const int u = u0 + i * NT; r[i] = Vec<T>::load(x + (size_t)(u < u_end ? u : u_end - 1) * VN); }
                    }
#pragma unroll
                    for (int i = 0; i < U; ++i) { const int u = u0 + i * NT; if (u < u_end) put(r[i], u); }
                }
            }
            if (tid < tail) g[nvec * VN + tid] = (T)(todo == ROW_COMPUTE ? cf * exp_gradient<T>(a, last - mr) : fill);
            team_sync();
            if (lead && todo == ROW_COMPUTE) {
                const double scale = exp_of(-log_z), ip = 1.0 / psum;
                for (int k = tid; k < a.K; k += LEAD) if (cls[k] >= 0) {
                    if (MODE == SPLIT && !(cls[k] / VN >= u_begin && cls[k] / VN < u_end) && !(tail > 0 && cls[k] >= nvec * VN)) continue;   // another slice's
                    const double q = ek[k] * scale;
                    const double d = a.reverse ? (q != 0.0 ? q * (log_of(ek[k]) - log_z - tk[k] - kl) : 0.0) : total * q - pk[k] * ip;
                    g[cls[k]] = (T)(acc)(a.tau * w * d);
                }
            }
        }
        // the bits back to 0 for the next row (a padded or wrong index has set none)
        if (lead && row + stride < a.n && w != 0.0) {
            wave_sync();
            for (int k = tid; k < a.K; k += LEAD) {
                const int64_t c = a.index_64 ? static_cast<const int64_t*>(a.index)[row * a.ld_index + k] : static_cast<const int32_t*>(a.index)[row * a.ld_index + k];
                if (c >= 0 && c < a.V) bits[c >> 5] = 0;
            }
        }
        team_sync();
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

template <typename T, int NT, int NV, int MODE = HELD> static int distill_run(hipStream_t stream, const DistillDev& d) {
    constexpr int ROWS = NT < 256 ? 256 / NT : 1;
    const size_t lds = distill_lds(d.V, d.K, NT) * ROWS;
    auto kernel = distill_kernel<T, NT, NV, MODE>;
    if (lds > 64 * 1024) OAK_CHECK(ensure_dynamic_lds((const void*)kernel, 160 * 1024));
    if constexpr (MODE == SPLIT) {
        const size_t bits = ((size_t)d.slice * Vec<T>::N + Vec<T>::N + 31) / 32 * 4;
        OAK_CHECK(launch(distill_slice_kernel<T, NT>, dim3((unsigned)d.slices, (unsigned)d.n), dim3(NT), bits, stream, d));
        return launch(kernel, dim3(d.dlogits ? (unsigned)d.slices : 1u, (unsigned)d.n), dim3(NT), lds, stream, d);
    }
    // a launch has fewer than 2^32 threads; the kernel walks on from row to row
    const int64_t wgs = (d.n + ROWS - 1) / ROWS, most = (int64_t)1 << 22;
    return launch(kernel, dim3((unsigned)(wgs < most ? wgs : most)), dim3(NT < 256 ? 256 : NT), lds, stream, d);
}

// Rows so long and so few that compute units would idle are cut into slices: at most 64 (a wave joins them), of at least 512 units,
// together at most two workgroups a compute unit.  With the gradient, one launch against two: 2 x 131072 bf16 24.8 -> 9.9 us, 64 x 131072
// 25.9 -> 15.0, 8 x 32768 11.3 -> 9.9, but 64 x 32768 11.7 -> 11.6, 8 x 16384 9.3 -> 9.8 and, in two slices, 200 x 131072 34.4 -> 38.6; the value
// alone is half of that work, and the second launch costs the host 3 us: from 8192 units on, for both, so that they agree to the last bit.
static int distill_slices(int64_t n, int V, int dtype) {
    const int64_t units = V / (16 / (int64_t)dtype_size(dtype));
    if (n <= 0 || n > 128 || units < 8192) return 1;
    int64_t s = 512 / n;
    if (s > 64) s = 64;
    if (s > units / 512) s = units / 512;
    return (int)s;
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
        const int units = (d.V + Vec<T>::N - 1) / Vec<T>::N;
        // the smallest team whose registers hold the row; few rows, with compute units to spare, are faster with many threads each
        // (8 rows of 32768 bf16: 11.2 us with 512 threads, 13.1 with 256)
        d.slices = distill_slices(d.n, d.V, a->dtype);
        const int whole = d.V / Vec<T>::N;
        if (d.slices > 1) {
            d.slice = (whole + d.slices - 1) / d.slices;
            d.slices = (whole + d.slice - 1) / d.slice;
            d.part = (double*)a->workspace;
            return distill_run<T, 512, 1, SPLIT>(stream, d);
        }
        if (d.n <= 256 && units > 64) return distill_run<T, 512, 8, LONG>(stream, d);
        constexpr int FEWEST = Vec<T>::N > 4 ? 8 : 4;              // as many threads as elements may be left over behind the units
        if (units <= 16 && d.K <= 16) return distill_run<T, FEWEST, 16 / FEWEST>(stream, d);
        if (units <= 64 && d.K <= 64) return distill_run<T, 16, 4>(stream, d);
        if (units <= 128 && d.K <= 64) return distill_run<T, 16, 8>(stream, d);
        if (units <= 256 && d.K <= 32) return distill_run<T, 16, 16>(stream, d);       // 65536 x 1000 float32: k = 10 120 us, with 64 threads 138;
        if (units <= 256) return distill_run<T, 64, 4>(stream, d);                     //   k = 64 237 us, with 64 threads 174
        if (units <= 512) return distill_run<T, 64, 8>(stream, d);
        if (units <= 1024) return distill_run<T, 64, 16>(stream, d);
        if (units <= 2048) return distill_run<T, 256, 8>(stream, d);
        if (units <= 4096) return distill_run<T, 256, 16>(stream, d);                  // 4096 x 32768 bf16: 117 us (4.6 TB/s), read twice 146
        // Longer rows: what 512 threads can hold with two workgroups a compute unit, the rest is read twice, the second time out of the last cache
        // (2 x 256 rows in flight fit it up to 2^18 bf16 classes, and the gradient passes it by).  2048 x 131072 bf16: 241 us (265 when this was
        // chosen; all of it read twice 279; the whole row in the registers of 1024 threads, one workgroup a unit, 330).
        return distill_run<T, 512, 8, LONG>(stream, d);
    });
}

}  // namespace oak

using namespace oak;

extern "C" {

int oak_device_pointer_check(oak_ctx* ctx, const void* p) {
    return c_entry([&] {
        OAK_REQUIRE(ctx != nullptr, "ctx is NULL");
        OAK_REQUIRE(p != nullptr, "the pointer is NULL");
        hipPointerAttribute_t at{};
        const hipError_t e = hipPointerGetAttributes(&at, p);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            OAK_REQUIRE(false, "%p is not memory of this library's HIP runtime (%s)", p, hipGetErrorString(e));
        }
        OAK_REQUIRE((at.type == hipMemoryTypeDevice || at.type == hipMemoryTypeManaged) && at.device == ctx->device,
                    "%p is not memory of device %d known to this library's HIP runtime", p, ctx->device);
        return (int)OAK_OK;
    });
}

int64_t oak_distill_workspace(oak_ctx* ctx, int64_t n_rows, int32_t n_classes, int32_t dtype) {
    if (!ctx || n_rows <= 0 || n_classes <= 0 || dtype < OAK_F64 || dtype > OAK_F16) return 0;
    const int slices = distill_slices(n_rows, n_classes, dtype);
    return slices > 1 ? n_rows * slices * 2 : 0;
}

int oak_distill_device(oak_ctx* ctx, void* stream, const oak_distill_args* a) {
    return c_entry([&] {
        OAK_CHECK(distill_check(a));
        const int64_t doubles = oak_distill_workspace(ctx, a->n_rows, a->n_classes, a->dtype);
        OAK_REQUIRE(doubles == 0 || (a->workspace && a->workspace_doubles >= doubles), "distill: the workspace holds %lld of the %lld doubles asked for by "
                    "oak_distill_workspace", (long long)a->workspace_doubles, (long long)doubles);
        DeviceGuard g;
        OAK_CHECK(g.enter(ctx));
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
        a.workspace_doubles = oak_distill_workspace(ctx, a.n_rows, a.n_classes, a.dtype);
        void* ws = nullptr;
        OAK_CHECK(get_buf(ctx, "kd_ws", (size_t)a.workspace_doubles * 8, &ws));
        a.workspace = (double*)ws;
        OAK_CHECK(distill_launch(ctx->stream, &a));
        t.stop();
        return st.finish();
    });
}

}  // extern "C"
