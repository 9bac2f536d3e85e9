// Mixtures of models: rows routed to their experts, laid out by expert, and the experts' answers summed with the router's weights.
//
//   route      x[n, e] -> the k experts of each row and their weights            (route_kernel), and the gradient (route_grad_kernel)
//   plan       experts[n, k] -> a stable order of the slots by expert             (plan_small_kernel | plan_count_piece / _join | plan_count / _scan / _place)
//   dispatch   X[n] copied to the places of its slots                              (dispatch_kernel)
//   combine    y[n] = sum_j w[n, j] F[place(n, j)], and its gradients              (combine_kernel, combine_grad_kernel)
//
// A hard assignment of rows (k-means labels) is the case k = 1 without a router.
#include "lowp.h"

namespace oak {

constexpr int64_t MOST_SLOTS = ((int64_t)1 << 31) - 1;      // places and slots are 32-bit numbers

// ---------------------------------------------------------------------------------------------------------------------
// route
// ---------------------------------------------------------------------------------------------------------------------
// A row belongs to a team of L lanes; lane l of the team holds the experts [l VPL, (l + 1) VPL) in registers, so that the row is read
// once, in pieces of VPL consecutive scores; a closed score is -inf from there on.  The k best are taken one after the other, lane j of
// the team keeps the j-th (L >= k).
//
// Keys.  Where nothing is added to the scores the keys are the scores themselves: softmax and sigmoid keep their order, and no rounding
// can tie what differs.  With a bias, or group scores that add two probabilities, the keys are probabilities in 64 bits: scores next to
// each other differ by less than the rounding of 32 bits often enough to matter (a few rows in ten thousand).
// A key carries its expert in its last bits, in the order that makes the larger key the lower expert, so that one maximum finds
// both and ties resolve themselves:
//   KEY_16   16-bit scores: a 31-bit integer, the score's bits in ascending order over 12 bits that no such score uses.  The next best after m
//            is the largest of key - m modulo 2^32: what is below m wraps to the upper half, and nothing has to be struck out
//   KEY_TAG  float scores and probabilities: a double whose last 11 of 52 bits are the tag (float scores do not reach them;
//            probabilities closer than 2^-41 of their size count as tied)
//   KEY_F64  double scores: all bits belong to the key, the expert is found in a second step
// Bound by the issue of vector instructions, 4 cycles each (counted: 0.9 of the time), not by memory.
enum { KEY_16 = 0, KEY_TAG = 1, KEY_F64 = 2 };

struct RouteDev {
    int64_t row0, n, ld, ld_mask, ld_out;
    int E, k, groups, top_groups, group_size, lanes_per_group;
    int dtype, sigmoid, top2, renorm, bias_f64;
    double scale;
    const void* scores; const void* bias; const unsigned char* mask;
    int* experts; void* weights;
    const void* dweights; void* dscores;
};

// A lane's piece of a row.  No branch depends on the lane: what lies behind the row's end is read from inside the row and replaced, so
// that all loads of a piece are in flight together (a branch around each would wait for its own).
template <typename T, int VPL, typename A> __device__ __forceinline__ void load_pieces(const T* p, int base, int E, A (&x)[VPL], A out_of_range) {
    if ((E & 3) == 0) {
        typedef T four __attribute__((ext_vector_type(4)));
        typedef four four_at __attribute__((aligned(sizeof(T))));
        four b[VPL / 4];
#pragma unroll
        for (int c = 0; c < VPL / 4; ++c) {
            const int e = base + 4 * c < E ? base + 4 * c : E - 4;
            b[c] = *reinterpret_cast<const four_at*>(p + e);
        }
#pragma unroll
        for (int s = 0; s < VPL; ++s) x[s] = base + (s & ~3) < E ? (A)b[s / 4][s & 3] : out_of_range;
    } else {
        T b[VPL];
#pragma unroll
        for (int s = 0; s < VPL; ++s) b[s] = p[base + s < E ? base + s : E - 1];
#pragma unroll
        for (int s = 0; s < VPL; ++s) x[s] = base + s < E ? (A)b[s] : out_of_range;
    }
}
// the lane's piece of a row of scores; the element type is a uniform branch: one kernel serves all of a kind
template <int VPL> __device__ __forceinline__ void load_scores(const RouteDev& a, int64_t row, int base, float (&x)[VPL]) {
    if (a.dtype == OAK_BF16) load_pieces<__bf16, VPL>(static_cast<const __bf16*>(a.scores) + row * a.ld, base, a.E, x, -INFINITY);
    else if (a.dtype == OAK_F16) load_pieces<_Float16, VPL>(static_cast<const _Float16*>(a.scores) + row * a.ld, base, a.E, x, -INFINITY);
    else load_pieces<float, VPL>(static_cast<const float*>(a.scores) + row * a.ld, base, a.E, x, -INFINITY);
}
template <int VPL> __device__ __forceinline__ void load_scores(const RouteDev& a, int64_t row, int base, double (&x)[VPL]) {
    load_pieces<double, VPL>(static_cast<const double*>(a.scores) + row * a.ld, base, a.E, x, (double)-INFINITY);
}
template <typename A> __device__ __forceinline__ A score_at(const RouteDev& a, int64_t row, int e) { return (A)load_any(a.scores, a.dtype, row * a.ld + e); }

// sigmoid; far below 0 (|x| > 700) what is left is 1e-304
__device__ __forceinline__ double sigmoid_of(double x) { return inverse(1.0 + exp_of(x < -700.0 ? 700.0 : -x)); }

// the piece with its masked scores closed (-inf); true if an open one of the row is NaN or +inf
template <int L, int VPL, typename A> __device__ __forceinline__ bool open_scores(const RouteDev& a, int64_t row, int base, A (&x)[VPL]) {
    if (a.mask != nullptr) {
        unsigned char m[VPL];
        load_pieces<unsigned char, VPL, unsigned char>(a.mask + row * a.ld_mask, base, a.E, m, 0);
        load_scores<VPL>(a, row, base, x);
#pragma unroll
        for (int s = 0; s < VPL; ++s) x[s] = m[s] != 0 ? x[s] : (A)-INFINITY;
    } else load_scores<VPL>(a, row, base, x);
    bool wrong = false;
#pragma unroll
    for (int s = 0; s < VPL; ++s) wrong |= !(x[s] < (A)INFINITY);
    return lanes_reduce<L>(wrong ? 1u : 0u, OpOr()) != 0;
}

// expert l VPL + s <-> tag: larger for lower experts
constexpr unsigned TAG_BITS = 2047;
__device__ __forceinline__ unsigned lane_tag(int l) { return (unsigned)(63 - l) << 5; }
template <int VPL> __device__ __forceinline__ int expert_of(unsigned tag) { return (63 - (int)(tag >> 5)) * VPL + 31 - (int)(tag & 31); }

// 16-bit scores
__device__ __forceinline__ unsigned key16(float x, unsigned lane, int s) {
    const unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);                          // -0 is 0
    const unsigned up = (b ^ ((unsigned)((int)b >> 31) | 0x80000000u)) >> 1;
    return (up & ~0xfffu) | lane | (unsigned)(31 - s);
}
constexpr unsigned KEY16_OPEN = 0x00800000u >> 1;                                       // the lowest finite score; -inf is below
__device__ __forceinline__ float key16_score(unsigned key) {
    const unsigned up = (key & ~0xfffu) << 1;
    return __builtin_bit_cast(float, up & 0x80000000u ? up ^ 0x80000000u : ~(up | 0x1fffu));
}

// float scores and probabilities; closed and struck keys have the high word of the lowest double
constexpr unsigned CLOSED_HI = 0xffefffffu;
constexpr double CLOSED_BELOW = -1.79e308;
__device__ __forceinline__ double with_hi(double v, unsigned hi) {
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | (unsigned)__builtin_bit_cast(unsigned long long, v));
}
__device__ __forceinline__ unsigned hi_of(double v) { return (unsigned)(__builtin_bit_cast(unsigned long long, v) >> 32); }
__device__ __forceinline__ double key_tagged(double x, unsigned lane, int s) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, x + 0.0);
    const unsigned sign = (unsigned)((int)(unsigned)(b >> 32) >> 31);                   // a larger magnitude is a smaller negative number
    const unsigned lo = ((unsigned)b & ~TAG_BITS) | ((lane | (unsigned)(31 - s)) ^ (sign & TAG_BITS));
    return __builtin_bit_cast(double, b >> 32 << 32 | lo);
}
__device__ __forceinline__ unsigned tag_of(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    return ((unsigned)b ^ (unsigned)((int)(unsigned)(b >> 32) >> 31)) & TAG_BITS;
}

// Maximum and minimum of a lane's own keys.  fmax() first quietens operands that may be signalling NaN (v_max_f64 of a register with itself),
// half of a selection's instructions where keys are put together from bits.  The results go to data-parallel moves first, never straight to
// a row swap, whose wait after an instruction of inline assembly is not the compiler's concern.
__device__ __forceinline__ double key_max(double a, double b) { double r; asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b)); return r; }
__device__ __forceinline__ double key_min(double a, double b) { double r; asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b)); return r; }
__device__ __forceinline__ float key_max(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ float key_min(float a, float b) { return __builtin_fminf(a, b); }

template <int KIND, int L, int VPL>
__global__ void __launch_bounds__(256) route_kernel(RouteDev a) {
    using acc = std::conditional_t<KIND == KEY_F64, double, float>;
    constexpr int TEAMS = 64 / L;
    extern __shared__ __align__(16) unsigned char lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, team = lane / L, l = lane & (L - 1);
    const int64_t row = a.row0 + ((int64_t)blockIdx.x * 4 + wave) * TEAMS + team, at = row < a.n ? row : a.n - 1;
    const int base = l * VPL;

    acc x[VPL];
    bool bad = open_scores<L, VPL>(a, at, base, x);

    // the softmax's maximum and sum, where something asks for them
    const bool plain_keys = KIND == KEY_16 || (a.bias == nullptr && !(a.groups > 1 && a.top2));
    acc xmax = 0, z = 0;
    if (!a.sigmoid && (!a.renorm || !plain_keys)) {
        xmax = x[0];
#pragma unroll
        for (int s = 1; s < VPL; ++s) xmax = OpMax()(xmax, x[s]);
        xmax = lanes_reduce<L>(xmax, OpMax());
        if (!a.renorm) {
#pragma unroll
            for (int s = 0; s < VPL; ++s) z += exp_of(x[s] - xmax);
            z = lanes_reduce<L>(z, OpSum());
        }
    }

    // keys without their tags: what groups are ranked by
    using clean = std::conditional_t<KIND == KEY_16, float, double>;
    clean v[VPL];
#pragma unroll
    for (int s = 0; s < VPL; ++s) v[s] = (clean)x[s];
    if constexpr (KIND != KEY_16) if (!plain_keys) {
        if (a.sigmoid) {
#pragma unroll
            for (int s = 0; s < VPL; ++s) v[s] = sigmoid_of((double)x[s]);
        } else {
            double zz = 0.0;
#pragma unroll
            for (int s = 0; s < VPL; ++s) { v[s] = exp_of((double)x[s] - (double)xmax); zz += x[s] == -INFINITY ? 0.0 : v[s]; }
            const double inv = inverse(lanes_reduce<L>(zz, OpSum()));
#pragma unroll
            for (int s = 0; s < VPL; ++s) v[s] *= inv;
        }
        if (a.bias != nullptr) {
            double b[VPL];
            if (a.bias_f64) load_pieces<double, VPL>(static_cast<const double*>(a.bias), base, a.E, b, 0.0);
            else load_pieces<float, VPL>(static_cast<const float*>(a.bias), base, a.E, b, 0.0);
            double odd = 0.0;                             // NaN if an entry is infinite or NaN: one instruction a score finds out
#pragma unroll
            for (int s = 0; s < VPL; ++s) { v[s] += b[s]; odd = __builtin_fma(b[s], 0.0, odd); }
            if (__any(odd != odd)) {
                // -inf closes its expert, NaN and +inf are like such a score (a tag would turn an infinite key into NaN)
                bool wrong = false;
#pragma unroll
                for (int s = 0; s < VPL; ++s) {
                    const double t = base + s >= a.E ? 0.0 : load_any(a.bias, a.bias_f64 ? OAK_F64 : OAK_F32, base + s);
                    wrong |= x[s] > (acc)-INFINITY && !(t < INFINITY);
                    if (t == -INFINITY) x[s] = -INFINITY;
                }
                bad |= lanes_reduce<L>(wrong ? 1u : 0u, OpOr()) != 0;
            }
        }
    }
    // a closed key: -inf, but for tags the lowest double (-inf with a tag would be NaN); scores of 64 bits reach that one themselves
    constexpr clean CLOSED = KIND == KEY_TAG ? (clean)-1.7976931348623157e308 : (clean)-INFINITY;
    auto is_open = [](clean t) { return t > (KIND == KEY_TAG ? (clean)CLOSED_BELOW : (clean)-INFINITY); };
#pragma unroll
    for (int s = 0; s < VPL; ++s) {
        if constexpr (KIND == KEY_TAG) v[s] = with_hi(v[s], x[s] == -INFINITY ? CLOSED_HI : hi_of(v[s]));
        else if constexpr (KIND == KEY_F64) v[s] = x[s] == -INFINITY ? CLOSED : v[s];
    }

    if (a.groups > 1) {
        clean* gs = reinterpret_cast<clean*>(lds) + (size_t)(wave * TEAMS + team) * (a.lanes_per_group ? a.groups : a.E + a.groups);
        if (a.lanes_per_group) {
            // a group is the whole of lanes_per_group neighbouring lanes: its two best by lane, then across them
            clean m1 = CLOSED, m2 = CLOSED;
#pragma unroll
            for (int s = 0; s < VPL; ++s) {
                m2 = key_max(m2, key_min(v[s], m1));
                m1 = key_max(m1, v[s]);
            }
            auto join = [&](auto mc) {
                constexpr int M = decltype(mc)::value;
                if constexpr (M < L) {
                    if (M < a.lanes_per_group) {
                        const clean o1 = lane_swap<M>(m1), o2 = lane_swap<M>(m2);
                        m2 = OpMax()(OpMax()(m2, o2), OpMin()(o1, m1));
                        m1 = OpMax()(m1, o1);
                    }
                }
            };
            join(std::integral_constant<int, 1>()); join(std::integral_constant<int, 2>()); join(std::integral_constant<int, 4>());
            join(std::integral_constant<int, 8>()); join(std::integral_constant<int, 16>()); join(std::integral_constant<int, 32>());
            const int g = l / a.lanes_per_group;
            const clean mine = a.top2 && is_open(m2) ? m1 + m2 : m1;
            if (g < a.groups) gs[g] = mine;
            wave_sync();
            int ahead = 0;
            for (int h = 0; h < a.groups; ++h) { const clean o = gs[h]; ahead += o > mine || (o == mine && h < g) ? 1 : 0; }
            if (ahead >= a.top_groups) {
#pragma unroll
                for (int s = 0; s < VPL; ++s) v[s] = CLOSED;
            }
        } else {
            // any other size: the team's keys through LDS, lane l scores the groups l, l + L, ...
            clean* keys = gs + a.groups;
#pragma unroll
            for (int s = 0; s < VPL; ++s) if (base + s < a.E) keys[base + s] = v[s];
            wave_sync();
            for (int g = l; g < a.groups; g += L) {
                clean m1 = CLOSED, m2 = CLOSED;
                for (int i = 0; i < a.group_size; ++i) {
                    const clean t = keys[g * a.group_size + i];
                    m2 = key_max(m2, key_min(t, m1));
                    m1 = key_max(m1, t);
                }
                gs[g] = a.top2 && is_open(m2) ? m1 + m2 : m1;
            }
            wave_sync();
            unsigned long long kept = 0;
            for (int g = l; g < a.groups; g += L) {
                const clean mine = gs[g];
                int ahead = 0;
                for (int h = 0; h < a.groups; ++h) { const clean o = gs[h]; ahead += o > mine || (o == mine && h < g) ? 1 : 0; }
                if (ahead < a.top_groups) kept |= 1ull << g;
            }
            kept = lanes_reduce<L>(kept, OpOr());
            int g = base / a.group_size, r = base - g * a.group_size;
#pragma unroll
            for (int s = 0; s < VPL; ++s) {
                if (g < a.groups && !(kept >> g & 1)) v[s] = CLOSED;
                if (++r == a.group_size) { r = 0; ++g; }
            }
        }
    }

    if constexpr (KIND != KEY_16) if (!plain_keys && a.bias == nullptr) {
        // probabilities were for the groups; the experts are chosen by the scores, which do not saturate
#pragma unroll
        for (int s = 0; s < VPL; ++s) v[s] = is_open(v[s]) ? (clean)x[s] : CLOSED;
    }

    // the k best; lane j of the team keeps the j-th and, where the key is the score, that
    int mine = -1;
    double xe = 0.0;
    if constexpr (KIND == KEY_F64) {
        for (int j = 0; j < a.k; ++j) {
            double m = CLOSED;
#pragma unroll
            for (int s = 0; s < VPL; ++s) m = v[s] > m ? v[s] : m;
            m = lanes_reduce<L>(m, OpMax());
            int best = a.E;
#pragma unroll
            for (int s = VPL - 1; s >= 0; --s) best = v[s] == m ? base + s : best;
            best = lanes_reduce<L>(best, OpMin());
#pragma unroll
            for (int s = 0; s < VPL; ++s) v[s] = base + s == best ? CLOSED : v[s];
            if (l == j) mine = is_open(m) ? best : -1;
        }
    } else if constexpr (KIND == KEY_16) {
        const unsigned tag = lane_tag(l);
        unsigned key[VPL], m = 0x80000000u, kept = 0;
#pragma unroll
        for (int s = 0; s < VPL; ++s) key[s] = key16(v[s], tag, s);
        for (int j = 0; j < a.k; ++j) {
            unsigned below = 0;
#pragma unroll
            for (int s = 0; s < VPL; ++s) below = OpMax()(below, key[s] - m);
            m += lanes_reduce<L>(below, OpMax());
            kept = l == j ? m : kept;
        }
        if (kept >= KEY16_OPEN) { mine = expert_of<VPL>(kept & TAG_BITS); xe = (double)key16_score(kept); }
    } else {
        const unsigned tag = lane_tag(l);
        double kept = CLOSED;
#pragma unroll
        for (int s = 0; s < VPL; ++s) v[s] = key_tagged(v[s], tag, s);
        for (int j = 0; j < a.k; ++j) {
            double m = v[0];
#pragma unroll
            for (int s = 1; s < VPL; ++s) m = key_max(m, v[s]);
            m = lanes_reduce<L>(m, OpMax());
#pragma unroll
            for (int s = 0; s < VPL; ++s) v[s] = with_hi(v[s], v[s] == m ? CLOSED_HI : hi_of(v[s]));
            kept = l == j ? m : kept;
        }
        if (is_open(kept)) { mine = expert_of<VPL>(tag_of(kept)); xe = __builtin_bit_cast(double, __builtin_bit_cast(long long, kept) & ~(long long)TAG_BITS); }
    }
    if (bad) mine = -1;

    // weights: one slot a lane, in 64 bits except for the plain softmax (a sigmoid's sum may be far below 1)
    const bool chosen = mine >= 0;
    if (chosen && (KIND == KEY_F64 || a.bias != nullptr)) xe = (double)score_at<acc>(a, at, mine);
    acc w = 0;
    if (a.renorm) {
        const double top = lanes_reduce<L>(chosen ? xe : -INFINITY, OpMax());
        // below -40 a sigmoid is the exponential to 2^-57
        double p = 0.0;
        if (chosen) p = a.sigmoid && top > -40.0 ? sigmoid_of(xe) : exp_of(xe - top);
        const double sum = lanes_reduce<L>(p, OpSum());
        if (chosen) w = (acc)(a.scale * (p / sum));               // a division: one expert's weight is 1 and not next to it
    } else if (chosen) {
        w = a.sigmoid ? (acc)(a.scale * (xe < -700.0 ? exp_of(xe) : sigmoid_of(xe))) : (acc)a.scale * (exp_of((acc)xe - xmax) / z);
    }
    if (row < a.n && l < a.k) {
        a.experts[row * a.k + l] = mine;
        static_cast<acc*>(a.weights)[row * a.k + l] = bad ? (acc)NAN : w;
    }
}

// d(scores).  With p = softmax or sigmoid, g_j = scale dw_j of the chosen and r their renormalised weights (without the scale):
//   softmax, plain   p_i (g_i [chosen] - sum_j p_j g_j)          sigmoid, plain   p_i (1 - p_i) g_i
//   softmax, renorm  r_i (g_i - sum_j r_j g_j)                    sigmoid, renorm  r_i (g_i - sum_j r_j g_j)(1 - p_i)
// Only the first is dense.  The chosen ones' terms go through an LDS row so that every row leaves in one coalesced piece; the dense one
// takes its dot product over that row too, so that no load waits for the experts' numbers (65536 x 160 bf16, k = 6: 14.6 us, 15.8 with
// the chosen scores read by number).  A row without experts has gradient zero.
template <typename A, int VPL, typename T> __device__ __forceinline__ void store_pieces(T* p, int base, int E, const A (&x)[VPL]) {
    typedef T four __attribute__((ext_vector_type(4)));
    typedef four four_at __attribute__((aligned(sizeof(T))));
#pragma unroll
    for (int c = 0; c < VPL; c += 4) {
        if (base + c + 4 <= E) {
            four b;
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = (T)x[c + i];
            *reinterpret_cast<four_at*>(p + base + c) = b;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (base + c + i < E) p[base + c + i] = (T)x[c + i];
        }
    }
}

template <typename acc, int L, int VPL>
__global__ void __launch_bounds__(256) route_grad_kernel(RouteDev a) {
    constexpr int TEAMS = 64 / L;
    extern __shared__ __align__(16) unsigned char lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, team = lane / L, l = lane & (L - 1);
    const int64_t row = a.row0 + ((int64_t)blockIdx.x * 4 + wave) * TEAMS + team;
    const bool live = row < a.n;
    const int64_t at = live ? row : a.n - 1;
    const int base = l * VPL;
    acc* buf = reinterpret_cast<acc*>(lds) + (size_t)(wave * TEAMS + team) * (L * VPL);
    const bool dense = !a.sigmoid && !a.renorm;

    // this lane's slot (L >= k); both loads on their way before either is looked at
    const int64_t slot = at * a.k + (l < a.k ? l : 0);
    const int e_read = a.experts[slot];
    const acc dw = static_cast<const acc*>(a.dweights)[slot];
    acc x[VPL], out[VPL];
    if (dense) {
        open_scores<L, VPL>(a, at, base, x);
    } else {
#pragma unroll
        for (int s = 0; s < VPL; ++s) x[s] = 0;
    }
#pragma unroll
    for (int s = 0; s < VPL; ++s) buf[base + s] = 0;
    const int e = l < a.k ? e_read : -1;
    const bool chosen = e >= 0 && e < a.E;
    const acc g = chosen ? (acc)a.scale * dw : (acc)0;
    const bool some = lanes_reduce<L>(chosen ? 1u : 0u, OpMax()) != 0;
    wave_sync();
    if (dense) {
        // every element against its g, 0 for what was not chosen
        if (chosen) atomicAdd(&buf[e], g);
        acc xmax = x[0];
#pragma unroll
        for (int s = 1; s < VPL; ++s) xmax = OpMax()(xmax, x[s]);
        xmax = lanes_reduce<L>(xmax, OpMax());
        acc z = 0;
#pragma unroll
        for (int s = 0; s < VPL; ++s) { x[s] = exp_of(x[s] - xmax); z += x[s]; }
        wave_sync();
        acc dot = 0;
#pragma unroll
        for (int s = 0; s < VPL; ++s) { out[s] = buf[base + s]; dot += x[s] * out[s]; }
        const acc inv = inverse(lanes_reduce<L>(z, OpSum()));
        dot = lanes_reduce<L>(dot, OpSum()) * inv;
#pragma unroll
        for (int s = 0; s < VPL; ++s) out[s] = some ? x[s] * inv * (out[s] - dot) : (acc)0;
    } else {
        const acc xe = chosen ? score_at<acc>(a, at, e) : (acc)0;
        const acc xmax = lanes_reduce<L>(chosen ? xe : (acc)-INFINITY, OpMax());
        acc r = 0, not_p = 1;
        if (a.sigmoid) {
            const acc p = (acc)1 / ((acc)1 + exp(-xe));        // sigmoid and 1 - sigmoid, each to its own size
            not_p = (acc)1 / ((acc)1 + exp(xe));
            if (chosen) r = !a.renorm || xmax > (acc)-40 ? p : exp_of(xe - xmax);
        } else if (chosen) r = exp_of(xe - xmax);
        if (a.renorm) r /= lanes_reduce<L>(r, OpSum());        // one expert's r is 1, its gradient 0
        const acc dot = lanes_reduce<L>(r * g, OpSum());
        if (chosen) atomicAdd(&buf[e], (a.renorm ? r * (g - dot) : r * g) * not_p);
        wave_sync();
#pragma unroll
        for (int s = 0; s < VPL; ++s) out[s] = buf[base + s];
    }
    if (!live) return;
    if constexpr (sizeof(acc) == 8) store_pieces<acc, VPL>(static_cast<double*>(a.dscores) + row * a.ld_out, base, a.E, out);
    else if (a.dtype == OAK_BF16) store_pieces<acc, VPL>(static_cast<__bf16*>(a.dscores) + row * a.ld_out, base, a.E, out);
    else if (a.dtype == OAK_F16) store_pieces<acc, VPL>(static_cast<_Float16*>(a.dscores) + row * a.ld_out, base, a.E, out);
    else store_pieces<acc, VPL>(static_cast<float*>(a.dscores) + row * a.ld_out, base, a.E, out);
}

// Lanes of a team and scores a lane.  Fewest lanes first, at most `most` scores each: the steps across lanes, which a row pays k
// times, and the work per row and wave are then fewest (kernel time: 1048576 x 24 float32, k = 2: 49 us with 4 lanes of 8, 27 with 2 of 12; 65536 x 160 bf16, k = 6:
// 17.5 us with 8 lanes of 24, 15.8 with 8 of 20; the gradient of those, which goes through LDS, 14.6 us with 16 of 12, 16.5 with 8 of 20, so
// that it stays at 16 scores a lane).  At least k lanes, so that every slot has one, and more of them while the rows fill less than 4 waves a
// SIMD and a lane has more than 4 scores: one row of 64 takes 2.4 us with 16 lanes, 3.1 with 8.
template <int MOST, typename F> static int with_team(int E, int k, int64_t rows, F&& fn) {
    auto by_vpl = [&](auto lc) {
        constexpr int L = decltype(lc)::value;
        const int per = (E + L - 1) / L;
        if (per <= 4) return fn(lc, std::integral_constant<int, 4>());
        if (per <= 8) return fn(lc, std::integral_constant<int, 8>());
        if (per <= 12) return fn(lc, std::integral_constant<int, 12>());
        if constexpr (MOST > 16) {
            if (per > 20) return fn(lc, std::integral_constant<int, 24>());
            if (per > 16) return fn(lc, std::integral_constant<int, 20>());
        }
        return fn(lc, std::integral_constant<int, 16>());
    };
    int lanes = 2;
    while (lanes < k || lanes * MOST < E) lanes *= 2;
    while (lanes < 64 && lanes * 4 < E && rows * lanes < (int64_t)64 * 4096) lanes *= 2;
    switch (lanes) {
        case 2: return by_vpl(std::integral_constant<int, 2>());
        case 4: return by_vpl(std::integral_constant<int, 4>());
        case 8: return by_vpl(std::integral_constant<int, 8>());
        case 16: return by_vpl(std::integral_constant<int, 16>());
        case 32: return by_vpl(std::integral_constant<int, 32>());
        default: return by_vpl(std::integral_constant<int, 64>());
    }
}

static int route_check(const oak_route_args* a) {
    OAK_REQUIRE(a != nullptr, "route: arguments are NULL");
    OAK_REQUIRE(a->n_rows >= 0, "route: n_rows = %lld", (long long)a->n_rows);
    OAK_REQUIRE(a->n_experts >= 1 && a->n_experts <= OAK_MAX_EXPERTS, "route: n_experts = %d is not in 1 .. %d", a->n_experts, OAK_MAX_EXPERTS);
    OAK_REQUIRE(a->n_groups >= 1 && a->n_groups <= 64 && a->n_experts % a->n_groups == 0,
                "route: n_groups = %d must divide the %d experts and be at most 64", a->n_groups, a->n_experts);
    OAK_REQUIRE(a->top_groups >= 1 && a->top_groups <= a->n_groups, "route: top_groups = %d of %d groups", a->top_groups, a->n_groups);
    OAK_REQUIRE(a->top_k >= 1 && a->top_k <= OAK_MAX_TOP_K && a->top_k <= a->top_groups * (a->n_experts / a->n_groups),
                "route: top_k = %d, at most %d and at most the experts of the groups kept (%d)", a->top_k, OAK_MAX_TOP_K,
                a->top_groups * (a->n_experts / a->n_groups));
    OAK_REQUIRE(a->dtype >= OAK_F64 && a->dtype <= OAK_F16, "route: unknown element type %d", a->dtype);
    OAK_REQUIRE(a->score == OAK_SCORE_SOFTMAX || a->score == OAK_SCORE_SIGMOID, "route: unknown score %d", a->score);
    OAK_REQUIRE(a->group_score == OAK_GROUP_MAX || a->group_score == OAK_GROUP_TOP2, "route: unknown group score %d", a->group_score);
    OAK_REQUIRE(a->scale - a->scale == 0.0, "route: scale is not finite");
    OAK_REQUIRE(a->n_rows <= 1 || (a->ld_scores >= 0 && (!a->mask || a->ld_mask >= 0)), "route: negative row stride");
    OAK_REQUIRE(a->n_rows == 0 || (a->scores && a->experts), "route: scores or experts are NULL");
    OAK_REQUIRE(a->n_rows <= MOST_SLOTS / a->top_k, "route: %lld rows x %d experts pass 2^31 slots", (long long)a->n_rows, a->top_k);
    return OAK_OK;
}

static RouteDev route_dev(const oak_route_args* a) {
    RouteDev d{};
    d.n = a->n_rows; d.ld = a->ld_scores; d.ld_mask = a->ld_mask; d.ld_out = a->ld_dscores;
    d.E = a->n_experts; d.k = a->top_k; d.groups = a->n_groups; d.top_groups = a->top_groups; d.group_size = a->n_experts / a->n_groups;
    d.sigmoid = a->score == OAK_SCORE_SIGMOID; d.top2 = a->group_score == OAK_GROUP_TOP2; d.dtype = a->dtype; d.renorm = a->renormalise != 0; d.bias_f64 = a->bias_f64;
    d.scale = a->scale; d.scores = a->scores; d.bias = a->bias; d.mask = a->mask; d.experts = a->experts; d.weights = a->weights;
    d.dweights = a->dweights; d.dscores = a->dscores;
    return d;
}

// a launch has fewer than 2^32 threads: more rows than 2^23 workgroups of 256 take are done in several
template <typename Args> static int launch_rows(void (*kernel)(Args), int rows_per_wg, size_t lds, hipStream_t stream, Args& d) {
    const int64_t most = (int64_t)rows_per_wg << 23;
    for (d.row0 = 0; d.row0 < d.n; d.row0 += most) {
        const int64_t rows = d.n - d.row0 < most ? d.n - d.row0 : most;
        OAK_CHECK(launch(kernel, dim3((unsigned)((rows + rows_per_wg - 1) / rows_per_wg)), dim3(256), lds, stream, d));
    }
    return OAK_OK;
}

static int route_launch(hipStream_t stream, const oak_route_args* a) {
    if (a->n_rows == 0) return OAK_OK;
    RouteDev d = route_dev(a);
    const bool plain_keys = d.bias == nullptr && !(d.groups > 1 && d.top2);
    auto run = [&](auto kind, auto most) {
        return with_team<decltype(most)::value>(d.E, d.k, d.n, [&](auto lc, auto vc) {
            constexpr int L = decltype(lc)::value, VPL = decltype(vc)::value, TEAMS = 64 / L;
            // groups that are whole lanes, a power of two of them, are scored without LDS
            const int lanes = d.group_size % VPL == 0 ? d.group_size / VPL : 0;
            d.lanes_per_group = lanes > 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
            const size_t lds = d.groups > 1 ? (size_t)4 * TEAMS * (d.lanes_per_group ? d.groups : d.E + d.groups) * sizeof(double) : 0;
            auto kernel = route_kernel<decltype(kind)::value, L, VPL>;
            if (lds > 64 * 1024) OAK_CHECK(ensure_dynamic_lds((const void*)kernel, 160 * 1024));
            return launch_rows(kernel, 4 * TEAMS, lds, stream, d);
        });
    };
    // 64-bit keys take twice the registers: at most 16 a lane
    if (d.dtype == OAK_F64) return run(std::integral_constant<int, KEY_F64>(), std::integral_constant<int, 16>());
    if (d.dtype != OAK_F32 && plain_keys) return run(std::integral_constant<int, KEY_16>(), std::integral_constant<int, 24>());
    return run(std::integral_constant<int, KEY_TAG>(), std::integral_constant<int, 16>());
}

static int route_grad_launch(hipStream_t stream, const oak_route_args* a) {
    if (a->n_rows == 0) return OAK_OK;
    RouteDev d = route_dev(a);
    return with_team<16>(d.E, d.k, d.n, [&](auto lc, auto vc) {
        constexpr int L = decltype(lc)::value, VPL = decltype(vc)::value, TEAMS = 64 / L;
        auto go = [&](auto zero) {
            using acc = decltype(zero);
            const size_t lds = (size_t)4 * TEAMS * L * VPL * sizeof(acc);
            return launch_rows(route_grad_kernel<acc, L, VPL>, 4 * TEAMS, lds, stream, d);
        };
        return d.dtype == OAK_F64 ? go((double)0) : go((float)0);
    });
}

// ---------------------------------------------------------------------------------------------------------------------
// plan: stable counting sort of the n k slots by expert
// ---------------------------------------------------------------------------------------------------------------------
// Bound by latency, two or three short launches (524288 slots, 24 experts: 12 us for 6 MB).  Every wave owns one consecutive piece of the
// slots, so that the order inside an expert is the slots' own without any atomic whose order could show: pieces are counted, the counts
// are summed in piece order, and each wave then places its slots 64 at a time -- a slot's rank among the 64 is the number of lower lanes
// with the same expert (one ballot per bit of the expert's number).  The experts of 4 such steps are asked for together (8000000 slots of 16
// experts: 58.6 us, one at a time 81.4).
constexpr int64_t PLAN_SMALL_SLOTS = 16384;
constexpr int PLAN_MAX_PIECES = 2048;
// two launches instead of three up to here: 524288 slots of 24 experts 11.9 us (three: 12.6), 20000 of 8 7.2 (9.7), and 2.5 us less of the host;
// 196608 slots of 64 experts 13.5 (11.5), 8000000 of 16 65.8 (58.6)
constexpr int PLAN_JOIN_EXPERTS = 32, PLAN_JOIN_PIECES = 512;
constexpr int64_t PLAN_JOIN_SLOTS = 1 << 20;

struct PlanDev {
    int64_t slots, piece;
    int k, E, npieces, bits;
    const int* experts; int* rows; int* positions; int* counts; int* offsets;
    int* ws;                    // [E][npieces]
};

// the experts of the slots s, s + STEP, ... below end (s may be behind it, end > 0), asked for together
template <int U, int STEP> __device__ __forceinline__ void slot_experts(const PlanDev& a, int64_t s, int64_t end, int (&e)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i) e[i] = a.experts[s + i * STEP < end ? s + i * STEP : end - 1];
#pragma unroll
    for (int i = 0; i < U; ++i) e[i] = s + i * STEP < end && (unsigned)e[i] < (unsigned)a.E ? e[i] : -1;      // whatever is not an expert's number belongs to no expert
}

// adds the slots [s0, s1) to cnt[e] (LDS), STEP threads of which this is number t
template <int STEP> __device__ __forceinline__ void plan_count_slots(const PlanDev& a, int* cnt, int64_t s0, int64_t s1, int t) {
    constexpr int U = 4;
    for (int64_t s = s0; s < s1; s += U * STEP) {
        int e[U];
        slot_experts<U, STEP>(a, s + t, s1, e);
#pragma unroll
        for (int i = 0; i < U; ++i) if (e[i] >= 0) atomicAdd(&cnt[e[i]], 1);
    }
}

// places the slots [s0, s1) of one wave; next[e] (LDS, this wave's own): where the expert's next slot goes
__device__ __forceinline__ void plan_place_piece(const PlanDev& a, int* next, int64_t s0, int64_t s1) {
    const int lane = threadIdx.x & 63;
    constexpr int U = 4;
    for (int64_t t = s0; t < s1; t += U * 64) {
        int es[U];
        slot_experts<U, 64>(a, t + lane, s1, es);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t s = t + i * 64 + lane;
            if (t + i * 64 >= s1) break;
            const int e = es[i];
            unsigned long long same = __ballot(e >= 0);
            for (int b = 0; b < a.bits; ++b) {
                const unsigned long long ones = __ballot(e >> b & 1);
                same &= (e >> b & 1) ? ones : ~ones;
            }
            int pos = -1;
            if (e >= 0) {
                const int rank = __popcll(same & (((unsigned long long)1 << lane) - 1));
                pos = next[e] + rank;
            }
            wave_sync();
            if (e >= 0 && (same >> lane) == 1ull) next[e] = pos + 1;      // the last of them
            wave_sync();
            if (s < s1) a.positions[s] = pos;
            if (pos >= 0) a.rows[pos] = (int)((unsigned)s / (unsigned)a.k);
        }
    }
}

// few slots: one workgroup of 16 waves does it all (one launch instead of three)
__global__ void __launch_bounds__(1024) plan_small_kernel(PlanDev a) {
    extern __shared__ int plan_lds[];                 // [16][E]
    int* cnt = plan_lds;
    __shared__ int wsum[17];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (int i = tid; i < 16 * a.E; i += 1024) cnt[i] = 0;
    __syncthreads();
    const int64_t s0 = wave * a.piece < a.slots ? wave * a.piece : a.slots, s1 = s0 + a.piece < a.slots ? s0 + a.piece : a.slots;
    plan_count_slots<64>(a, cnt + wave * a.E, s0, s1, lane);
    __syncthreads();
    int total = 0;                                    // E <= 1024: one expert per thread
    if (tid < a.E) for (int w = 0; w < 16; ++w) total += cnt[w * a.E + tid];
    int incl = total;
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(incl, d, 64); if (lane >= d) incl += o; }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int off = incl - total, all = 0;
    for (int w = 0; w < 16; ++w) { if (w < wave) off += wsum[w]; all += wsum[w]; }
    if (tid < a.E) {
        a.counts[tid] = total; a.offsets[tid] = off;
        for (int w = 0; w < 16; ++w) { const int c = cnt[w * a.E + tid]; cnt[w * a.E + tid] = off; off += c; }
    }
    if (tid == 0) a.offsets[a.E] = all;
    __syncthreads();
    plan_place_piece(a, cnt + wave * a.E, s0, s1);
    for (int64_t s = all + tid; s < a.slots; s += 1024) a.rows[s] = -1;
}

__global__ void __launch_bounds__(256) plan_count_kernel(PlanDev a) {
    extern __shared__ int plan_lds[];                 // [4][E]
    int* cnt = plan_lds;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t piece = (int64_t)blockIdx.x * 4 + wave;
    int* mine = cnt + wave * a.E;
    for (int e = lane; e < a.E; e += 64) mine[e] = 0;
    wave_sync();
    const int64_t s0 = piece * a.piece, s1 = s0 + a.piece < a.slots ? s0 + a.piece : a.slots;
    plan_count_slots<64>(a, mine, s0, s1, lane);
    wave_sync();
    if (piece < a.npieces) for (int e = lane; e < a.E; e += 64) a.ws[(int64_t)e * a.npieces + piece] = mine[e];
}

// one workgroup per expert: counts of its pieces -> what lies before each piece
__global__ void __launch_bounds__(256) plan_scan_kernel(PlanDev a) {
    __shared__ int wsum[4];
    const int e = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int* col = a.ws + (int64_t)e * a.npieces;
    constexpr int PER = PLAN_MAX_PIECES / 256;
    int c[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { c[i] = tid * PER + i < a.npieces ? col[tid * PER + i] : 0; mine += c[i]; }
    int incl = mine;
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(incl, d, 64); if (lane >= d) incl += o; }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int before = incl - mine;
    for (int w = 0; w < wave; ++w) before += wsum[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) { if (tid * PER + i < a.npieces) col[tid * PER + i] = before; before += c[i]; }
    if (tid == 255) a.counts[e] = before;
}

__global__ void __launch_bounds__(256) plan_place_kernel(PlanDev a) {
    extern __shared__ int plan_lds[];                 // [4][E] next places, [E + 1] offsets
    int* lds = plan_lds;
    __shared__ int wsum[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int* off = lds + 4 * a.E;
    // offsets of the experts from their counts: every workgroup sums them itself
    const int per = (a.E + 255) / 256, e0 = tid * per, e1 = e0 + per < a.E ? e0 + per : a.E;
    int mine = 0;
    for (int e = e0; e < e1; ++e) mine += a.counts[e];
    int incl = mine;
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(incl, d, 64); if (lane >= d) incl += o; }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int at = incl - mine;
    for (int w = 0; w < wave; ++w) at += wsum[w];
    for (int e = e0; e < e1; ++e) { off[e] = at; at += a.counts[e]; }
    if (tid == 0) off[a.E] = wsum[0] + wsum[1] + wsum[2] + wsum[3];
    __syncthreads();
    if (blockIdx.x == 0) for (int e = tid; e <= a.E; e += 256) a.offsets[e] = off[e];
    const int all = off[a.E];
    const int64_t piece = (int64_t)blockIdx.x * 4 + wave;
    if (piece < a.npieces) {
        int* next = lds + wave * a.E;
        for (int e = lane; e < a.E; e += 64) next[e] = off[e] + a.ws[(int64_t)e * a.npieces + piece];
        wave_sync();
        const int64_t s0 = piece * a.piece, s1 = s0 + a.piece < a.slots ? s0 + a.piece : a.slots;
        plan_place_piece(a, next, s0, s1);
        for (int64_t s = s0 + lane; s < s1; s += 64) if (s >= all) a.rows[s] = -1;
    }
}

// Few experts: the counts of 512 pieces, a workgroup each, ...
__global__ void __launch_bounds__(256) plan_count_piece_kernel(PlanDev a) {
    __shared__ int cnt[PLAN_JOIN_EXPERTS];
    const int tid = threadIdx.x;
    if (tid < a.E) cnt[tid] = 0;
    __syncthreads();
    const int64_t s0 = blockIdx.x * a.piece, s1 = s0 + a.piece < a.slots ? s0 + a.piece : a.slots;
    plan_count_slots<256>(a, cnt, s0, s1, tid);
    __syncthreads();
    if (tid < a.E) a.ws[(int64_t)tid * a.npieces + blockIdx.x] = cnt[tid];
}

// ... which every workgroup sums itself (wave w the experts w, w + 4, ...) before each of its waves places a quarter of its piece
__global__ void __launch_bounds__(256) plan_join_kernel(PlanDev a) {
    __shared__ int cnt[4][64], next[4][PLAN_JOIN_EXPERTS], before[PLAN_JOIN_EXPERTS], total[PLAN_JOIN_EXPERTS];
    static_assert(PLAN_JOIN_EXPERTS <= 64, "a lane an expert");
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, piece = (int)blockIdx.x;
    const int64_t end = (piece + 1) * a.piece < a.slots ? (piece + 1) * a.piece : a.slots, quarter = a.piece / 4;
    const int64_t q0 = piece * a.piece + wave * quarter, s0 = q0 < end ? q0 : end, s1 = s0 + quarter < end ? s0 + quarter : end;
    cnt[wave][lane] = 0;
    wave_sync();
    plan_count_slots<64>(a, cnt[wave], s0, s1, lane);
    constexpr int U = 4;                              // columns asked for together
    for (int e0 = wave; e0 < a.E; e0 += 4 * U) {
        int c[U][PLAN_JOIN_PIECES / 64];
#pragma unroll
        for (int q = 0; q < U; ++q) {
            const int* col = a.ws + (int64_t)(e0 + 4 * q < a.E ? e0 + 4 * q : e0) * a.npieces;
#pragma unroll
            for (int i = 0; i < PLAN_JOIN_PIECES / 64; ++i) c[q][i] = i * 64 + lane < a.npieces ? col[i * 64 + lane] : 0;
        }
#pragma unroll
        for (int q = 0; q < U; ++q) {
            int mine = 0, all = 0;
#pragma unroll
            for (int i = 0; i < PLAN_JOIN_PIECES / 64; ++i) { all += c[q][i]; mine += i * 64 + lane < piece ? c[q][i] : 0; }
            mine = lanes_reduce<64>(mine, OpSum());
            all = lanes_reduce<64>(all, OpSum());
            if (lane == 0 && e0 + 4 * q < a.E) { before[e0 + 4 * q] = mine; total[e0 + 4 * q] = all; }
        }
    }
    __syncthreads();
    const int mine = lane < a.E ? total[lane] : 0;
    int incl = mine;
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(incl, d, 64); if (lane >= d) incl += o; }
    const int off = incl - mine, all = __shfl(incl, 63, 64);
    if (lane < a.E) {
        int at = off + before[lane];
        for (int w = 0; w < wave; ++w) at += cnt[w][lane];
        next[wave][lane] = at;
        if (piece == 0 && wave == 0) { a.counts[lane] = mine; a.offsets[lane] = off; }
    }
    if (piece == 0 && threadIdx.x == 0) a.offsets[a.E] = all;
    wave_sync();
    plan_place_piece(a, next[wave], s0, s1);
    for (int64_t s = s0 + lane; s < s1; s += 64) if (s >= all) a.rows[s] = -1;
}

enum { PLAN_SMALL = 0, PLAN_JOIN = 1, PLAN_SCAN = 2 };

static int plan_pieces(int64_t slots, int E, int64_t* piece, int* npieces) {
    const int kind = slots <= PLAN_SMALL_SLOTS && E <= 1024 ? PLAN_SMALL : E <= PLAN_JOIN_EXPERTS && slots <= PLAN_JOIN_SLOTS ? PLAN_JOIN : PLAN_SCAN;
    // PLAN_SCAN: 8 waves a compute unit; with many experts fewer, so that the table of counts stays within 2^20 integers
    const int want = kind == PLAN_SMALL ? 16 : kind == PLAN_JOIN ? PLAN_JOIN_PIECES : E <= 512 ? PLAN_MAX_PIECES : (1 << 20) / E;
    const int64_t step = kind == PLAN_JOIN ? 256 : 64, least = kind == PLAN_SMALL ? 64 : 256;
    int64_t p = (slots + want - 1) / want;
    p = p < least ? least : (p + step - 1) / step * step;
    *piece = p;
    *npieces = (int)((slots + p - 1) / p);
    return kind;
}

static int64_t plan_workspace(int64_t n_rows, int32_t top_k, int32_t n_experts) {
    if (n_rows <= 0 || top_k <= 0 || n_experts <= 0 || n_experts > OAK_MAX_PLAN_EXPERTS || n_rows > MOST_SLOTS / top_k) return 0;
    int64_t piece; int np;
    return plan_pieces(n_rows * top_k, n_experts, &piece, &np) == PLAN_SMALL ? 0 : (int64_t)np * n_experts;
}

static int plan_check(const oak_plan_args* a) {
    OAK_REQUIRE(a != nullptr, "plan: arguments are NULL");
    OAK_REQUIRE(a->n_rows >= 0 && a->top_k >= 1 && a->top_k <= OAK_MAX_TOP_K, "plan: %lld rows of %d experts", (long long)a->n_rows, a->top_k);
    OAK_REQUIRE(a->n_experts >= 1 && a->n_experts <= OAK_MAX_PLAN_EXPERTS, "plan: n_experts = %d is not in 1 .. %d", a->n_experts, OAK_MAX_PLAN_EXPERTS);
    OAK_REQUIRE(a->n_rows <= MOST_SLOTS / a->top_k, "plan: %lld rows x %d experts pass 2^31 slots", (long long)a->n_rows, a->top_k);
    OAK_REQUIRE(a->counts && a->offsets && (a->n_rows == 0 || (a->experts && a->rows && a->positions)), "plan: an array is NULL");
    return OAK_OK;
}

static int plan_launch(hipStream_t stream, const oak_plan_args* a) {
    PlanDev d{};
    d.slots = a->n_rows * a->top_k; d.k = a->top_k; d.E = a->n_experts;
    const int kind = plan_pieces(d.slots, d.E, &d.piece, &d.npieces);
    d.experts = a->experts; d.rows = a->rows; d.positions = a->positions; d.counts = a->counts; d.offsets = a->offsets; d.ws = a->workspace;
    while ((1 << d.bits) < d.E) ++d.bits;
    if (kind == PLAN_SMALL) {
        const size_t lds = (size_t)16 * d.E * sizeof(int);
        if (lds > 32 * 1024) OAK_CHECK(ensure_dynamic_lds((const void*)plan_small_kernel, 16 * 1024 * sizeof(int)));
        return launch(plan_small_kernel, dim3(1), dim3(1024), lds, stream, d);
    }
    if (kind == PLAN_JOIN) {
        OAK_CHECK(launch(plan_count_piece_kernel, dim3((unsigned)d.npieces), dim3(256), 0, stream, d));
        return launch(plan_join_kernel, dim3((unsigned)d.npieces), dim3(256), 0, stream, d);
    }
    const unsigned wgs = (unsigned)((d.npieces + 3) / 4);
    const size_t lds = (size_t)(5 * d.E + 1) * sizeof(int);
    if (lds > 32 * 1024) {
        OAK_CHECK(ensure_dynamic_lds((const void*)plan_count_kernel, 128 * 1024));
        OAK_CHECK(ensure_dynamic_lds((const void*)plan_place_kernel, 128 * 1024));
    }
    OAK_CHECK(launch(plan_count_kernel, dim3(wgs), dim3(256), (size_t)4 * d.E * sizeof(int), stream, d));
    OAK_CHECK(launch(plan_scan_kernel, dim3((unsigned)d.E), dim3(256), 0, stream, d));
    return launch(plan_place_kernel, dim3(wgs), dim3(256), lds, stream, d);
}

// ---------------------------------------------------------------------------------------------------------------------
// dispatch, combine and their gradients
// ---------------------------------------------------------------------------------------------------------------------
// All of them walk rows: a row is read or written once where the slots' order would touch it k times.  tpr threads share a row; a unit is
// 16 bytes, the row's last elements that do not fill one are units of their own.  A thread asks for the places, then for the answers of up
// to 8 slots before it adds the first (k = 6: combine 198 us, 4 at a time 210).  Bound by memory: 32768 rows, k = 6, 2048 bf16 columns, of 0.94 GB
// each: dispatch 177 us (5.3 TB/s), combine 178 (5.3), and of 1.74 GB combine_grad 352 (4.9), where a large copy reaches 5.06 TB/s.
struct MixDev {
    int64_t row0, n, slots, ld_rows, ld_slots, ld_grad;
    int64_t units;              // 16-byte units of a row, then its last elements
    int C, k, nvec, E, tpr, inv_tpr, rows_per_wg, tpr_log2;
    const int* positions; const int* offsets; const void* weights;
    const void* src; void* dst; const void* dout; void* dslots; void* dweights;
};

template <typename T> __device__ __forceinline__ void zero_unit(const MixDev& a, T* row, int64_t u) {
    if (u < a.nvec) { typename Vec<T>::raw z = {}; Vec<T>::store(row + u * Vec<T>::N, z); }
    else row[a.nvec * (int64_t)Vec<T>::N + (u - a.nvec)] = (T)0;
}

// slots of 1 KiB and more are written past the caches (32768 x 2048 bf16, k = 6: all five calls of a training step 922 -> 899 us: dispatch
// 158 -> 177, but the combine that reads other slots meanwhile 198 -> 178; 262144 x 17
// float64, whose rows end inside cache lines, 88 -> 90)
template <typename T, bool WIDE> __device__ __forceinline__ void store_slot(T* p, typename Vec<T>::raw v) {
    if constexpr (WIDE) Vec<T>::store_stream(p, v); else Vec<T>::store(p, v);
}

// a place outside [0, slots) is no place
__device__ __forceinline__ int64_t place_of(const MixDev& a, int64_t n, int j) {
    const int p = a.positions[n * a.k + j];
    return p >= 0 && p < a.slots ? p : -1;
}

// row and first unit of this thread: 256 / tpr rows a workgroup, the threads left over have none (-1)
__device__ __forceinline__ int64_t mix_row(const MixDev& a, int* unit) {
    const int r = (int)(((unsigned)threadIdx.x * (unsigned)a.inv_tpr) >> 16);
    *unit = (int)threadIdx.x - r * a.tpr;
    const int64_t n = a.row0 + (int64_t)blockIdx.x * a.rows_per_wg + r;
    return r < a.rows_per_wg && n < a.n ? n : -1;
}

template <typename T, bool WIDE> __global__ void __launch_bounds__(256) dispatch_kernel(MixDev a) {
    int t;
    const int64_t n = mix_row(a, &t);
    if (n < 0) return;
    const T* src = static_cast<const T*>(a.src) + n * a.ld_rows;
    T* dst = static_cast<T*>(a.dst);
    const int used = a.offsets[a.E];
    for (int64_t u = t; u < a.units; u += a.tpr) {
        if (u < a.nvec) {
            const auto v = Vec<T>::load(src + u * Vec<T>::N);
            for (int j = 0; j < a.k; ++j) { const int64_t p = place_of(a, n, j); if (p >= 0) store_slot<T, WIDE>(dst + p * a.ld_slots + u * Vec<T>::N, v); }
        } else {
            const int64_t c = a.nvec * (int64_t)Vec<T>::N + (u - a.nvec);
            const T v = src[c];
            for (int j = 0; j < a.k; ++j) { const int64_t p = place_of(a, n, j); if (p >= 0) dst[p * a.ld_slots + c] = v; }
        }
        if (n * a.k + a.k > used)
            for (int j = 0; j < a.k; ++j) if (n * a.k + j >= used) zero_unit<T>(a, dst + (n * a.k + j) * a.ld_slots, u);
    }
}

template <typename T, int CHUNK> __global__ void __launch_bounds__(256) combine_kernel(MixDev a) {
    using acc = typename Num<T>::acc;
    int t;
    const int64_t n = mix_row(a, &t);
    if (n < 0) return;
    const T* src = static_cast<const T*>(a.src);
    T* dst = static_cast<T*>(a.dst) + n * a.ld_rows;
    const acc* w = static_cast<const acc*>(a.weights);
    for (int64_t u = t; u < a.units; u += a.tpr) {
        const bool whole = u < a.nvec;
        const int64_t c = whole ? u * Vec<T>::N : a.nvec * (int64_t)Vec<T>::N + (u - a.nvec);
        acc y[Vec<T>::N] = {};
        for (int j0 = 0; j0 < a.k; j0 += CHUNK) {
            int64_t p[CHUNK];
            acc wj[CHUNK];
            typename Vec<T>::raw f[CHUNK];
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) {
                p[i] = j0 + i < a.k ? place_of(a, n, j0 + i) : -1;
                wj[i] = j0 + i < a.k && w ? w[n * a.k + j0 + i] : (acc)(j0 + i < a.k);
            }
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) {
                const T* at = src + p[i] * a.ld_slots + c;
                f[i] = typename Vec<T>::raw{};
                if (p[i] >= 0) { if (whole) f[i] = Vec<T>::load(at); else f[i][0] = *at; }
            }
            // no expert: the weight times nothing (a NaN weight still shows)
#pragma unroll
            for (int i = 0; i < CHUNK; ++i)
#pragma unroll
                for (int e = 0; e < Vec<T>::N; ++e) y[e] += wj[i] * (acc)f[i][e];
        }
        if (whole) {
            typename Vec<T>::raw o;
#pragma unroll
            for (int e = 0; e < Vec<T>::N; ++e) o[e] = (T)y[e];
            Vec<T>::store(dst + c, o);
        } else dst[c] = (T)y[0];
    }
}

// dF[place] = w dy, dw = <dy, F[place]>: slot by slot, the row of dy stays in the nearest cache, 4 units of both asked for together.  At
// most 64 threads a row: the dot product is finished inside a wave.  It is 32 bits within a unit and 64 across units: one lane adds up to a
// 64th of a row, whose roundings all fall to one side where the row is flat (2^20 equal columns: 2e-4 of the sum in 32 bits).
template <typename T, bool WIDE> __global__ void __launch_bounds__(256) combine_grad_kernel(MixDev a) {
    using acc = typename Num<T>::acc;
    const int64_t n = a.row0 + (int64_t)blockIdx.x * a.rows_per_wg + (threadIdx.x >> a.tpr_log2);
    const int tpr = 1 << a.tpr_log2, t = (int)(threadIdx.x & (tpr - 1));
    const bool live = n < a.n;                         // whole waves stay for the shuffles
    const T* F = static_cast<const T*>(a.src);
    const T* dy = static_cast<const T*>(a.dout) + (live ? n : 0) * a.ld_grad;
    T* dF = static_cast<T*>(a.dslots);
    const acc* w = static_cast<const acc*>(a.weights);
    const int used = a.offsets[a.E];
    for (int j = 0; j < a.k; ++j) {
        const int64_t p = live ? place_of(a, n, j) : -1;
        double d = 0.0;
        if (p >= 0) {
            const acc wj = w[n * a.k + j];
            const T* fr = F + p * a.ld_slots;
            T* gr = dF + p * (int64_t)a.C;
            constexpr int U = 4;                       // units asked for together
            for (int64_t u0 = t; u0 < a.nvec; u0 += U * tpr) {
                typename Vec<T>::raw f[U], v[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int64_t u = u0 + i * tpr < a.nvec ? u0 + i * tpr : u0;
                    f[i] = Vec<T>::load(fr + u * Vec<T>::N);
                    v[i] = Vec<T>::load(dy + u * Vec<T>::N);
                }
#pragma unroll
                for (int i = 0; i < U; ++i) if (u0 + i * tpr < a.nvec) {
                    typename Vec<T>::raw o;
                    acc unit = 0;
#pragma unroll
                    for (int e = 0; e < Vec<T>::N; ++e) { unit += (acc)f[i][e] * (acc)v[i][e]; o[e] = (T)(wj * (acc)v[i][e]); }
                    d += (double)unit;
                    store_slot<T, WIDE>(gr + (u0 + i * tpr) * Vec<T>::N, o);
                }
            }
            for (int64_t c = (int64_t)a.nvec * Vec<T>::N + t; c < a.C; c += tpr) {
                const acc v = (acc)dy[c];
                d += (double)((acc)fr[c] * v);
                gr[c] = (T)(wj * v);
            }
        }
        for (int m = 1; m < tpr; m <<= 1) d += __shfl_xor(d, m, 64);
        if (live && t == 0) static_cast<acc*>(a.dweights)[n * a.k + j] = (acc)d;
        if (live && n * a.k + j >= used) for (int64_t u = t; u < a.units; u += tpr) zero_unit<T>(a, dF + (n * a.k + j) * (int64_t)a.C, u);
    }
}

static int mix_check(const char* what, const oak_mix_args* a) {
    OAK_REQUIRE(a != nullptr, "%s: arguments are NULL", what);
    OAK_REQUIRE(a->n_rows >= 0 && a->top_k >= 1 && a->top_k <= OAK_MAX_TOP_K, "%s: %lld rows of %d experts", what, (long long)a->n_rows, a->top_k);
    OAK_REQUIRE(a->n_experts >= 1 && a->n_experts <= OAK_MAX_PLAN_EXPERTS, "%s: n_experts = %d", what, a->n_experts);
    OAK_REQUIRE(a->n_cols >= 1 && a->n_cols <= (1 << 30), "%s: n_cols = %d", what, a->n_cols);
    OAK_REQUIRE(a->dtype >= OAK_F64 && a->dtype <= OAK_F16, "%s: unknown element type %d", what, a->dtype);
    OAK_REQUIRE(a->n_rows <= MOST_SLOTS / a->top_k, "%s: %lld rows x %d experts pass 2^31 slots", what, (long long)a->n_rows, a->top_k);
    OAK_REQUIRE(a->ld_rows >= 0 && a->ld_slots >= 0 && a->ld_grad >= 0, "%s: negative row stride", what);
    OAK_REQUIRE(a->n_rows == 0 || (a->positions && a->offsets), "%s: positions or offsets are NULL", what);
    return OAK_OK;
}

static int mix_launch(hipStream_t stream, const oak_mix_args* a, int what /* 0 dispatch, 1 combine, 2 combine_grad */) {
    if (a->n_rows == 0) return OAK_OK;
    MixDev d{};
    const int vec = 16 / (int)dtype_size(a->dtype);
    d.n = a->n_rows; d.k = a->top_k; d.slots = d.n * d.k; d.ld_rows = a->ld_rows; d.ld_slots = a->ld_slots; d.ld_grad = a->ld_grad; d.C = a->n_cols;
    d.E = a->n_experts; d.nvec = d.C / vec; d.units = d.nvec + d.C % vec;
    d.positions = a->positions; d.offsets = a->offsets; d.weights = a->weights; d.src = a->src; d.dst = a->dst; d.dout = a->dout;
    d.dslots = a->dslots; d.dweights = a->dweights;
    // combine_grad: a power of two within a wave; the others: as many threads as the row has units
    while (d.tpr_log2 < 6 && ((int64_t)1 << d.tpr_log2) < d.units) ++d.tpr_log2;
    d.tpr = d.units < 256 ? (int)d.units : 256;
    d.rows_per_wg = what == 2 ? 256 >> d.tpr_log2 : 256 / d.tpr;
    d.inv_tpr = (65536 + d.tpr - 1) / d.tpr;           // t / tpr = t inv_tpr >> 16 for t < 256
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        const bool wide = (int64_t)d.C * (int64_t)sizeof(T) >= 1024;
        auto kernel = what == 0 ? (wide ? dispatch_kernel<T, true> : dispatch_kernel<T, false>)
                      : what == 2 ? (wide ? combine_grad_kernel<T, true> : combine_grad_kernel<T, false>)
                      : d.k <= 2 ? combine_kernel<T, 2> : d.k <= 4 ? combine_kernel<T, 4> : combine_kernel<T, 8>;
        return launch_rows(kernel, d.rows_per_wg, 0, stream, d);
    });
}

}  // namespace oak

using namespace oak;

extern "C" {

int oak_route_device(oak_ctx* ctx, void* stream, const oak_route_args* a) {
    return c_entry([&] {
        OAK_CHECK(route_check(a));
        OAK_REQUIRE(a->n_rows == 0 || a->weights, "route: weights are NULL");
        DeviceGuard g;
        OAK_CHECK(g.enter(ctx));
        return route_launch((hipStream_t)stream, a);
    });
}

int oak_route_grad_device(oak_ctx* ctx, void* stream, const oak_route_args* a) {
    return c_entry([&] {
        OAK_CHECK(route_check(a));
        OAK_REQUIRE(a->n_rows == 0 || (a->dweights && a->dscores), "route_grad: dweights or dscores are NULL");
        OAK_REQUIRE(a->n_rows <= 1 || a->ld_dscores >= a->n_experts, "route_grad: rows of dscores overlap");
        DeviceGuard g;
        OAK_CHECK(g.enter(ctx));
        return route_grad_launch((hipStream_t)stream, a);
    });
}

static int route_host(oak_ctx* ctx, const oak_route_args* args, bool grad) {
    if (!ctx) { set_error("ctx is NULL"); return OAK_E_ARG; }
    OAK_CHECK(route_check(args));
    OAK_REQUIRE(args->dtype == OAK_F64 && (!args->bias || args->bias_f64), "route: host arrays are float64");
    OAK_REQUIRE(args->ld_scores == args->n_experts && (!args->mask || args->ld_mask == args->n_experts || args->ld_mask == 0),
                "route: host arrays are contiguous");
    OAK_REQUIRE(args->n_rows == 0 || (grad ? args->dweights && args->dscores && args->ld_dscores == args->n_experts : args->weights != nullptr),
                "route: an array is NULL");
    OAK_HIP_CHECK(hipSetDevice(ctx->device));
    if (args->n_rows == 0) return OAK_OK;
    PhaseTimer t(ctx, grad ? "route_grad" : "route");
    oak_route_args a = *args;
    HostStage st(ctx);
    const size_t cells = (size_t)a.n_rows * a.n_experts, slots = (size_t)a.n_rows * a.top_k;
    OAK_CHECK(st.in("ex_scores", a.scores, cells * 8));
    OAK_CHECK(st.in("ex_bias", a.bias, (size_t)a.n_experts * 8));
    OAK_CHECK(st.in("ex_mask", a.mask, a.ld_mask ? cells : (size_t)a.n_experts));
    if (grad) {
        OAK_CHECK(st.in("ex_experts", a.experts, slots * 4));
        OAK_CHECK(st.in("ex_dweights", a.dweights, slots * 8));
        OAK_CHECK(st.out("ex_dscores", a.dscores, cells * 8));
        OAK_CHECK(route_grad_launch(ctx->stream, &a));
    } else {
        OAK_CHECK(st.out("ex_experts", a.experts, slots * 4));
        OAK_CHECK(st.out("ex_weights", a.weights, slots * 8));
        OAK_CHECK(route_launch(ctx->stream, &a));
    }
    t.stop();
    return st.finish();
}

int oak_route(oak_ctx* ctx, const oak_route_args* a) { return c_entry([&] { return route_host(ctx, a, false); }); }
int oak_route_grad(oak_ctx* ctx, const oak_route_args* a) { return c_entry([&] { return route_host(ctx, a, true); }); }

int64_t oak_plan_workspace(oak_ctx* ctx, int64_t n_rows, int32_t top_k, int32_t n_experts) {
    return ctx ? plan_workspace(n_rows, top_k, n_experts) : 0;
}

int oak_plan_device(oak_ctx* ctx, void* stream, const oak_plan_args* a) {
    return c_entry([&] {
        OAK_CHECK(plan_check(a));
        const int64_t ints = plan_workspace(a->n_rows, a->top_k, a->n_experts);
        OAK_REQUIRE(ints == 0 || (a->workspace && a->workspace_ints >= ints), "plan: the workspace holds %lld of the %lld integers asked for by oak_plan_workspace",
                    (long long)a->workspace_ints, (long long)ints);
        DeviceGuard g;
        OAK_CHECK(g.enter(ctx));
        return plan_launch((hipStream_t)stream, a);
    });
}

int oak_plan(oak_ctx* ctx, const oak_plan_args* args) {
    return c_entry([&] {
        if (!ctx) { set_error("ctx is NULL"); return OAK_E_ARG; }
        OAK_CHECK(plan_check(args));
        OAK_HIP_CHECK(hipSetDevice(ctx->device));
        PhaseTimer t(ctx, "plan");
        oak_plan_args a = *args;
        HostStage st(ctx);
        const size_t slots = (size_t)a.n_rows * a.top_k;
        OAK_CHECK(st.in("ex_experts", a.experts, slots * 4));
        OAK_CHECK(st.out("ex_rows", a.rows, slots * 4));
        OAK_CHECK(st.out("ex_positions", a.positions, slots * 4));
        OAK_CHECK(st.out("ex_counts", a.counts, (size_t)a.n_experts * 4));
        OAK_CHECK(st.out("ex_offsets", a.offsets, (size_t)(a.n_experts + 1) * 4));
        a.workspace_ints = plan_workspace(a.n_rows, a.top_k, a.n_experts);
        void* ws = nullptr;
        OAK_CHECK(get_buf(ctx, "ex_plan_ws", (size_t)a.workspace_ints * 4, &ws));
        a.workspace = (int32_t*)ws;
        OAK_CHECK(plan_launch(ctx->stream, &a));
        t.stop();
        return st.finish();
    });
}

static int mix_arrays(const char* name, const oak_mix_args* a, int what) {
    OAK_CHECK(mix_check(name, a));
    if (a->n_rows == 0) return OAK_OK;
    OAK_REQUIRE(a->src != nullptr, "%s: the input is NULL", name);
    if (what == 2) {
        OAK_REQUIRE(a->weights && a->dout && a->dslots && a->dweights, "%s: an array is NULL", name);
    } else {
        OAK_REQUIRE(a->dst != nullptr, "%s: the output is NULL", name);
        const int64_t ld_out = what == 0 ? a->ld_slots : a->ld_rows;
        OAK_REQUIRE(a->n_rows * (what == 0 ? a->top_k : 1) <= 1 || ld_out >= a->n_cols, "%s: rows of the output overlap", name);
    }
    return OAK_OK;
}

static int mix_device(const char* name, oak_ctx* ctx, void* stream, const oak_mix_args* a, int what) {
    return c_entry([&] {
        OAK_CHECK(mix_arrays(name, a, what));
        DeviceGuard g;
        OAK_CHECK(g.enter(ctx));
        return mix_launch((hipStream_t)stream, a, what);
    });
}

static int mix_host(const char* name, oak_ctx* ctx, const oak_mix_args* args, int what) {
    return c_entry([&] {
        if (!ctx) { set_error("ctx is NULL"); return OAK_E_ARG; }
        OAK_CHECK(mix_arrays(name, args, what));
        OAK_REQUIRE(args->dtype == OAK_F64 && args->ld_rows == args->n_cols && args->ld_slots == args->n_cols && args->ld_grad == args->n_cols,
                    "%s: host arrays are contiguous float64", name);
        OAK_HIP_CHECK(hipSetDevice(ctx->device));
        if (args->n_rows == 0) return (int)OAK_OK;
        PhaseTimer t(ctx, name);
        oak_mix_args a = *args;
        HostStage st(ctx);
        const size_t slots = (size_t)a.n_rows * a.top_k, rb = (size_t)a.n_rows * a.n_cols * 8, sb = slots * a.n_cols * 8;
        OAK_CHECK(st.in("ex_positions", a.positions, slots * 4));
        OAK_CHECK(st.in("ex_offsets", a.offsets, (size_t)(a.n_experts + 1) * 4));
        OAK_CHECK(st.in("ex_weights", a.weights, slots * 8));
        if (what == 0) {
            OAK_CHECK(st.in("mix_rows", a.src, rb));
            OAK_CHECK(st.out("mix_slots", a.dst, sb));
        } else {
            OAK_CHECK(st.in("mix_slots", a.src, sb));
            if (what == 1) OAK_CHECK(st.out("mix_rows", a.dst, rb));
            else {
                OAK_CHECK(st.in("mix_rows", a.dout, rb));
                OAK_CHECK(st.out("mix_dslots", a.dslots, sb));
                OAK_CHECK(st.out("mix_dweights", a.dweights, slots * 8));
            }
        }
        OAK_CHECK(mix_launch(ctx->stream, &a, what));
        t.stop();
        return st.finish();
    });
}

int oak_dispatch(oak_ctx* ctx, const oak_mix_args* a) { return mix_host("dispatch", ctx, a, 0); }
int oak_combine(oak_ctx* ctx, const oak_mix_args* a) { return mix_host("combine", ctx, a, 1); }
int oak_combine_grad(oak_ctx* ctx, const oak_mix_args* a) { return mix_host("combine_grad", ctx, a, 2); }
int oak_dispatch_device(oak_ctx* ctx, void* stream, const oak_mix_args* a) { return mix_device("dispatch", ctx, stream, a, 0); }
int oak_combine_device(oak_ctx* ctx, void* stream, const oak_mix_args* a) { return mix_device("combine", ctx, stream, a, 1); }
int oak_combine_grad_device(oak_ctx* ctx, void* stream, const oak_mix_args* a) { return mix_device("combine_grad", ctx, stream, a, 2); }

}  // extern "C"
