// Distillation from a teacher's top logits (stes_distill / stes_distill_bwd in include/stes.h): the temperature-scaled KL divergence
// of the student's softmax over all V classes from the teacher's softmax over its k best, and its gradient.
//
// Everything is bound by the logits' trip through memory, so they are read once: a team of threads holds a row (or a lane group a
// short row) in registers as it was loaded, takes the maximum, the sum of exp, and writes q straight from the registers; the listed
// classes, k of V, are written over by the lanes that hold them.  Rows too long for a workgroup's registers are read twice (the
// second time mostly from the cache).
//
// Measured (a copy of 1 GiB runs at 4,980 GB/s): loss and gradient in one pass of 8,192 x 32,003 bf16 205 us (5.1 TB/s); of
// 2,048 x 50,001 fp32 loss 83 to 110 us and gradient 148 us (4.9 TB/s and, behind the gradient's writes, 3.7; 5.5 TB/s); 16,384 x 1,000
// bf16 17 and 15 us (bound by the teacher's part of a row, some 200 instructions a wave, and its chain of loads: index, then logit);
// short rows are bound by instructions too: 131,072 x 300 bf16 loss 55 us, gradient 57 us.
#include "stes_common.h"

namespace {

template <typename T, int V> struct Vec;
template <> struct Vec<bf16, 8> { typedef bf16x8 type; };
template <> struct Vec<float, 4> { typedef f32x4 type; };
template <typename T> struct Vec<T, 1> { typedef T type __attribute__((ext_vector_type(1))); };

// Everything is in base 2: the card's exp and log are.
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }

// v of another lane of the wave: CTRL names it as DPP does; lanes that have none, or whose row is not in ROWS, get `none`
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp(float none, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) {       // (every lane has a source)
    return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
constexpr int ROW_ROR = 0x120, ROW_SHR = 0x110, ROW_BCAST15 = 0x142, ROW_BCAST31 = 0x143;
constexpr int QUAD_XOR1 = 0xB1, QUAD_XOR2 = 0x4E, ROW_HALF_MIRROR = 0x141, ROW_MIRROR = 0x140;

// f over the G < 64 lanes of a lane group, the result in all of them.  (Once the lanes of a quad hold the same, mirroring eight lanes
// swaps its quads; likewise on.)
template <int G, typename F> __device__ __forceinline__ float group_fold(float v, F f) {
    v = f(v, dpp<QUAD_XOR1, 0xf>(v, v));
    v = f(v, dpp<QUAD_XOR2, 0xf>(v, v));
    if (G >= 8) v = f(v, dpp<ROW_HALF_MIRROR, 0xf>(v, v));
    if (G >= 16) v = f(v, dpp<ROW_MIRROR, 0xf>(v, v));
    if (G >= 32) v = f(v, __shfl_xor(v, 16, 64));
    return v;
}

// What another lane of this wave wrote to LDS is read next (a wave's LDS accesses are executed in order; this keeps the compiler's).
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// reductions over the G lanes of an aligned lane group
template <int G> __device__ __forceinline__ float group_max(float v) {
    if constexpr (G == 64) {                                 // (all lanes active; six DPP steps instead of six trips through LDS)
        constexpr float low = -INFINITY;
        v = fmaxf(v, dpp<ROW_SHR + 1, 0xf>(low, v));
        v = fmaxf(v, dpp<ROW_SHR + 2, 0xf>(low, v));
        v = fmaxf(v, dpp<ROW_SHR + 4, 0xf>(low, v));
        v = fmaxf(v, dpp<ROW_SHR + 8, 0xf>(low, v));
        v = fmaxf(v, dpp<ROW_BCAST15, 0xa>(low, v));
        v = fmaxf(v, dpp<ROW_BCAST31, 0xc>(low, v));
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
    }
    return group_fold<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G> __device__ __forceinline__ float group_sum(float v) {
    if constexpr (G == 64) {
        v += dpp<ROW_SHR + 1, 0xf>(0.f, v);
        v += dpp<ROW_SHR + 2, 0xf>(0.f, v);
        v += dpp<ROW_SHR + 4, 0xf>(0.f, v);
        v += dpp<ROW_SHR + 8, 0xf>(0.f, v);
        v += dpp<ROW_BCAST15, 0xa>(0.f, v);
        v += dpp<ROW_BCAST31, 0xc>(0.f, v);
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
    }
    return group_fold<G>(v, [](float a, float b) { return a + b; });
}
template <int G> __device__ __forceinline__ bool group_any(bool b, int lane) {
    const uint64_t m = __ballot(b);
    if (G == 64) return m != 0;
    return ((m >> (lane & ~(G - 1))) & ((1ull << (G & 63)) - 1)) != 0;
}

struct Entry {
    int at;                  // a listed class of the row; < 0: none in this lane
    float p;                 // its probability
    bool some, bad;          // of the row: it lists a class of some probability; it lists an index beyond V or a value that is no number
};

// a lane's value, from place j of the lane's group
template <int G> __device__ __forceinline__ int from(int v, int j, int lane) {
    return G == 64 ? __builtin_amdgcn_readlane(v, j) : __shfl(v, (lane & ~(G - 1)) + j, 64);
}
template <int G> __device__ __forceinline__ float from(float v, int j, int lane) { return __int_as_float(from<G>(__float_as_int(v), j, lane)); }

// a ^ b is zero where a key is found again N or fewer places further on in its row of 16 lanes, which closes into a ring
template <int N> struct Ring {
    static __device__ __forceinline__ unsigned nearest(unsigned a, unsigned b) {
        const unsigned here = a ^ dpp<ROW_ROR + N>(b), nearer = Ring<N - 1>::nearest(a, b);
        return here < nearer ? here : nearer;
    }
};
template <> struct Ring<0> { static __device__ __forceinline__ unsigned nearest(unsigned, unsigned) { return ~0u; } };

// Whether the lane's class is held by another lane of its group as well; of two lanes that share one at least one says so.  Half a ring
// of 16 holds every pair once; a group of more lanes compares its rows of 16 with one another.
template <int G>
__device__ __forceinline__ bool listed_twice(int at, int lane, int k) {
    const unsigned key = at < 0 ? 0x80000000u | (unsigned)lane : (unsigned)at ^ (G < 16 ? (unsigned)(lane / G) << 24 : 0u);
    unsigned d = Ring<(G < 8 ? G - 1 : G == 8 ? 7 : 8)>::nearest(key, key);
    if (G >= 32 && k > 16) {
#pragma unroll
        for (int o = 16; o < G; o += 16) {
            const unsigned other = (unsigned)__shfl_xor((int)key, o, 64), x = key ^ other, y = Ring<8>::nearest(key, other);
            d = min(d, min(x, y));
            if (o == 16 && k <= 32) break;
        }
    }
    return d == 0;
}

struct Listed { int at; float v; };      // one place of a row's list as it was loaded: index (< 0: unused, V: beyond the classes) and value

__device__ __forceinline__ Listed load_listed(const stes_distill_args& p, long m, bool row, int l) {
    Listed e{-1, -INFINITY};
    if (row && l < p.k) {
        const long o = m * p.ld_idx + l, i = p.idx_i64 ? ((const int64_t*)p.idx)[o] : (long)((const int32_t*)p.idx)[o];
        const long ov = m * p.ld_val + l;
        const float u = p.val_f32 ? ((const float*)p.val)[ov] : (float)((const bf16*)p.val)[ov];
        if (i >= 0) { e.at = i >= p.V ? p.V : (int)i; e.v = u; }
    }
    return e;
}

// The teacher's distribution of a row, an entry per lane of a group of G >= k lanes (`l`: the lane's place in it).  A class that is
// listed more than once has its whole probability at its first place; the later places hold none.  With entries == false only
// what the row is worth (some, bad) is found out.
template <int G>
__device__ __forceinline__ Entry teacher_row(const stes_distill_args& p, const Listed& in, int l, int lane, float ct, bool entries) {
    Entry e;
    e.at = in.at;
    const float v = in.v;
    const float mx = group_max<G>(v);                       // (fmaxf passes over NaN: those are caught below)
    e.bad = group_any<G>(e.at >= p.V || v != v || v == INFINITY, lane);
    e.some = mx > -INFINITY || e.bad;
    e.p = 0.f;
    if (!entries) {
        e.at = -1;
        return e;
    }
    float w = v > -INFINITY ? exp2_((v - mx) * ct) : 0.f;
    w *= __builtin_amdgcn_rcpf(group_sum<G>(w));
    // merge duplicates, which hardly ever occur
    float whole = w;
    int first = l;
    if (__any(listed_twice<G>(e.at, lane, p.k))) {
        whole = 0.f;
        first = G;
        for (int j = 0; j < p.k; ++j) {
            const int aj = from<G>(e.at, j, lane);
            const float pj = from<G>(w, j, lane);
            if (aj == e.at) { whole += pj; first = first < j ? first : j; }
        }
    }
    e.p = whole;
    if (first != l || !(whole >= 1.17549435e-38f) || e.at >= p.V) e.at = -1;       // (what is not a normal number counts as nothing)
    return e;
}

// the factor of a row's gradient; `scale` = grad_scale temperature / denom
__device__ __forceinline__ float row_factor(const stes_distill_args& p, float scale, float w, bool bad) {
    const float f = scale * w * (p.upstream ? p.upstream[0] : 1.f);
    return bad ? __builtin_nanf("") : f;
}

// A lane's part of KL tau / 4 = sum P (log P - log q) tau / 4, for a class of probability P and logit s; ls = log2(sum), tl = tau ln 2 / 4.
// Logits of the type's lowest value stay finite in it: nothing multiplies their distance from the maximum by more than 1.
__device__ __forceinline__ float kl_part(float P, float s, float mx, float ls, float tl) { return P * (tl * (log2_(P) + ls) - (0.25f * s - 0.25f * mx)); }

constexpr int MAX_ROUNDS = 1 << 22;                  // (an exit for broken zeros: the loss becomes NaN)

// A workgroup's part of the loss (`sum` is thread 0's, in 64 bits: rows near 3e38 may pass fp32's range together, before `factor` divides them);
// the only one of a launch is the loss.  With `p.zeros` the workgroups hand their parts to the last one, which adds them up in an order of its
// own: words that are valid when they are not zero (a part of 0 is 5e-324 instead), in relaxed atomics of agent scope, and it leaves them
// zero.  One workgroup waits and the others wait for nothing: every wait ends.  Without them, and from 16 parts a thread on, where reading
// them one after the other takes longer than a launch, distill_sum_kernel adds up.  Loss and gradient of 1,024 x 7 4.4 us (two launches
// 6.3, one workgroup in one launch 9.7), of 16,384 x 1,000 20.4 (21.1); loss of 30,000 x 600, 7,500 parts for 256 threads, 23.8 (22.6).
__host__ __device__ inline bool in_one_launch(const stes_distill_args& p, int blocks, int threads) {
    return blocks == 1 || (p.zeros && blocks <= STES_DISTILL_WORDS && blocks <= 16 * threads);
}

__device__ __forceinline__ uint64_t part_word(double sum) { const uint64_t w = (uint64_t)__double_as_longlong(sum); return w ? w : 1u; }

template <int BLOCK>
__device__ __forceinline__ void hand_over(const stes_distill_args& p, double sum, double factor, double* red) {
    if (gridDim.x == 1 || !in_one_launch(p, gridDim.x, BLOCK)) {
        if (threadIdx.x == 0) {
            if (gridDim.x == 1) *p.loss = (float)(sum * factor);
            else ((double*)p.ws)[blockIdx.x] = sum;
        }
        return;
    }
    const int n = gridDim.x - 1;
    if (blockIdx.x != n) {
        if (threadIdx.x == 0) __hip_atomic_store(p.zeros + blockIdx.x, part_word(sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return;
    }
    double s = threadIdx.x == 0 ? sum : 0.0;
    for (int i = threadIdx.x; i < n; i += 4 * BLOCK) {
        uint64_t w[4];
        bool all = false;
        for (int round = 0; !all && round < MAX_ROUNDS; ++round) {
            if (round) __builtin_amdgcn_s_sleep(4);
            all = true;
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = i + u * BLOCK < n ? __hip_atomic_load(p.zeros + i + u * BLOCK, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 1u;
#pragma unroll
            for (int u = 0; u < 4; ++u) all = all && w[u] != 0;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            s += all ? __longlong_as_double((long long)w[u]) : __builtin_nan("");
            if (i + u * BLOCK < n) __hip_atomic_store(p.zeros + i + u * BLOCK, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < BLOCK / 64; ++w) t += red[w];
        *p.loss = (float)(t * factor);
    }
}

enum { LOSS = 1, GRAD = 2, STATS_IN = 4 };           // what a launch does

// ---------------------------------------------------------------- short rows
// V <= E G and k <= G: a group of G lanes per row, at most E classes a lane, neighbouring lanes neighbouring classes.  BLOCK / G rows a
// workgroup and round, the next round's rows loaded ahead; a workgroup's rows follow from its index alone, and so does the order
// of its sum.
template <typename TS, int G, int E> struct ShortRow {
    TS x[E];
    Listed listed;
    float w;
    __device__ __forceinline__ void load(const stes_distill_args& p, long m, int l) {
        const bool row = m < p.M;
        const TS* s = (const TS*)p.logits + m * p.ld;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = row && e * G + l < p.V ? s[e * G + l] : (TS)0.f;
        w = row ? (p.weight ? p.weight[m] : 1.f) : 0.f;
        listed = load_listed(p, m, row, l);
    }
};

template <typename TS, typename TG, int G, int E, int BLOCK, int MODE>
__global__ __launch_bounds__(BLOCK) void distill_short_kernel(const stes_distill_args p, int rounds, double factor, float scale) {
    constexpr int RPB = BLOCK / G;
    __shared__ double red[BLOCK / 64];
    __shared__ float target[MODE & GRAD ? BLOCK * E : 1];    // P of the rows at work, zero but for the listed classes
    const int lane = threadIdx.x & 63, l = threadIdx.x % G;
    float* const mine = target + (MODE & GRAD ? threadIdx.x / G * (G * E) : 0);
    if (MODE & GRAD) {
#pragma unroll
        for (int e = 0; e < E; ++e) mine[e * G + l] = 0.f;
    }
    const float ct = LOG2E / p.temperature, tl = p.temperature * (0.25f * LN2);
    const long first = (long)blockIdx.x * rounds * RPB + threadIdx.x / G;
    double total = 0.0;
    ShortRow<TS, G, E> next;
    next.load(p, first, l);
    for (int r = 0; r < rounds; ++r) {
        const long m = first + r * RPB;
        const bool row = m < p.M;
        const ShortRow<TS, G, E> in = next;
        if (r + 1 < rounds) next.load(p, m + RPB, l);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = row && e * G + l < p.V ? (float)in.x[e] : -INFINITY;
        const float w = in.w;
        const Entry t = teacher_row<G>(p, in.listed, l, lane, ct, true);
        const bool counts = t.some && w != 0.f;
        float mx, sum;
        if (MODE & STATS_IN) { mx = row ? p.stats[2 * m] : 0.f; sum = row ? p.stats[2 * m + 1] : 1.f; }
        else {
            mx = x[0];
#pragma unroll
            for (int e = 1; e < E; ++e) mx = fmaxf(mx, x[e]);
            mx = group_max<G>(mx);
        }
        float q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = e * G + l < p.V ? exp2_((x[e] - mx) * ct) : 0.f;
        if (!(MODE & STATS_IN)) {
            sum = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) sum += q[e];
            sum = group_sum<G>(sum);
            if (p.stats && row && l == 0) { p.stats[2 * m] = mx; p.stats[2 * m + 1] = sum; }
        }
        if (MODE & LOSS) {
            const float st = t.at >= 0 ? (float)((const TS*)p.logits)[m * p.ld + t.at] : 0.f;
            float kl = group_sum<G>(t.at >= 0 ? kl_part(t.p, st, mx, log2_(sum), tl) : 0.f);
            if (t.bad) kl = __builtin_nanf("");
            if (counts && l == 0) total += (double)w * kl;
        }
        if (MODE & GRAD) {
            if (t.at >= 0) mine[t.at] = t.p;
            wave_lds_fence();
            if (row) {
                const float f = row_factor(p, scale, w, t.bad), inv = __builtin_amdgcn_rcpf(sum);
                TG* d = (TG*)p.dlogits + m * p.ld_d;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int v = e * G + l;
                    if (v < p.V) {
                        const float g = counts ? f * (q[e] * inv - mine[v]) : 0.f;
                        if (!p.accumulate) d[v] = (TG)g;
                        else if (counts) d[v] = (TG)((float)d[v] + g);
                    }
                }
            }
            wave_lds_fence();
            if (t.at >= 0) mine[t.at] = 0.f;
            wave_lds_fence();
        }
    }
    if (MODE & LOSS) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
        if (lane == 0) red[threadIdx.x >> 6] = total;
        __syncthreads();
        if (threadIdx.x == 0) {
            total = 0.0;
            for (int w = 0; w < BLOCK / 64; ++w) total += red[w];
        }
        hand_over<BLOCK>(p, total, factor, red);
    }
}

// ---------------------------------------------------------------- rows in registers
// A team of TEAM threads holds a row: N vectors of 16 bytes a thread (W elements each), a few elements in front of the first 16-byte
// boundary and behind the last one as single elements.  TEAM = 64: a wave per row, four rows a workgroup, no barrier.
// STREAM: rows of any length, read again instead of held.  Seven waves a SIMD for TEAM = 64: loss of 16,384 x 1,000 15.2 us, 16.4 with six.
template <int TEAM> struct Team {
    static constexpr int WAVES = TEAM / 64;
    static __device__ __forceinline__ float max_(float v, float* red) {
        v = group_max<64>(v);
        if (WAVES == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v = fmaxf(v, red[w]);
        return v;
    }
    static __device__ __forceinline__ float sum_(float v, float* red) {
        v = group_sum<64>(v);
        if (WAVES == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += red[w];
        return v;
    }
    static __device__ __forceinline__ void sync() {
        if (WAVES > 1) __syncthreads();
        else { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
    }
};

// f(i, row[i]) for i = i0, i0 + TEAM, ... below n, four loads in flight
template <int TEAM, typename VT, typename F>
__device__ __forceinline__ void walk(const VT* row, int i0, int n, F f) {
    int i = i0;
    for (; i + 3 * TEAM < n; i += 4 * TEAM) {
        VT y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = row[i + u * TEAM];
#pragma unroll
        for (int u = 0; u < 4; ++u) f(i + u * TEAM, y[u]);
    }
    for (; i < n; i += TEAM) f(i, row[i]);
}

template <typename TS, typename TG, int W, int TEAM, int N, bool STREAM, int MODE>
__global__ __launch_bounds__(TEAM == 64 ? 256 : TEAM, TEAM == 64 ? 7 : 1) void distill_row_kernel(const stes_distill_args p, double factor, float scale) {
    typedef typename Vec<TS, W>::type VS;
    typedef typename Vec<TG, W>::type VG;
    typedef Team<TEAM> Tm;
    constexpr int RPB = TEAM == 64 ? 4 : 1, BLOCK = TEAM * RPB;
    __shared__ float red[BLOCK / 64];
    __shared__ double parts[BLOCK / 64];
    const int lane = threadIdx.x & 63, i0 = threadIdx.x % TEAM;
    const long m = (long)blockIdx.x * RPB + threadIdx.x / TEAM;
    const bool row = m < p.M;
    double out = 0.0;
    if (row) {
        // (the list first: 8,192 x 32,003 bf16, 32 listed: loss 108 to 105 us, gradient 207 to 201, both 207 to 203.5)
        const Listed listed = load_listed(p, m, true, lane);
        const TS* s = (const TS*)p.logits + m * p.ld;
        const float ct = LOG2E / p.temperature;
        const float w = p.weight ? p.weight[m] : 1.f;
        const int V = p.V;
        // [0, head) single, then nv vectors, then [tail, V) single
        const int head = W == 1 ? 0 : min(V, (int)((16 - ((uintptr_t)s & 15)) & 15) / (int)sizeof(TS));
        const int nv = (V - head) / W, tail = head + nv * W, rest = V - tail;
        const VS* sv = reinterpret_cast<const VS*>(s + head);
        const int single = i0 < head ? i0 : (i0 - head < rest ? tail + i0 - head : -1);        // (head + rest < 2 W <= TEAM)
        VS x[STREAM ? 1 : N];
        float x1 = -INFINITY;
        if (W > 1 && single >= 0) x1 = (float)s[single];
        if (!STREAM) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i * TEAM + i0 < nv) x[i] = sv[i * TEAM + i0];
        }
        float st = 0.f;                                      // (asked for ahead of the work on the list)
        if (threadIdx.x % TEAM < 64 && listed.at >= 0 && listed.at < p.V) st = (float)s[listed.at];
        const Entry t = teacher_row<64>(p, listed, lane, lane, ct, threadIdx.x % TEAM < 64);
        const bool counts = t.some && w != 0.f;
        float mx = 0.f, sum = 1.f;
        if (MODE & STATS_IN) { mx = p.stats[2 * m]; sum = p.stats[2 * m + 1]; }
        else if (counts) {
            mx = x1;
            if (STREAM) {
                // running maximum and sum: a thread's sum is scaled when its maximum rises
                float acc = 0.f;
                auto take = [&](const VS& y) {
                    float top = (float)y[0];
#pragma unroll
                    for (int e = 1; e < W; ++e) top = fmaxf(top, (float)y[e]);
                    if (top > mx) { acc *= mx > -INFINITY ? exp2_((mx - top) * ct) : 0.f; mx = top; }
                    float add = 0.f;
                    if (mx > -INFINITY) {
#pragma unroll
                        for (int e = 0; e < W; ++e) add += exp2_(((float)y[e] - mx) * ct);
                    } else {                                 // -inf and NaN alone so far
#pragma unroll
                        for (int e = 0; e < W; ++e) add += (float)y[e] == -INFINITY ? 0.f : __builtin_nanf("");
                    }
                    acc += add;
                };
                walk<TEAM>(sv, i0, nv, [&](int, const VS& y) { take(y); });
                if (x1 > -INFINITY || x1 != x1) acc += exp2_((x1 - mx) * ct);
                const float own = mx;
                mx = Tm::max_(mx, red);
                sum = Tm::sum_(own > -INFINITY || acc != 0.f ? acc * exp2_((own - mx) * ct) : 0.f, red);
                if (mx == -INFINITY) sum = __builtin_nanf("");
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i * TEAM + i0 < nv)
#pragma unroll
                        for (int e = 0; e < W; ++e) mx = fmaxf(mx, (float)x[i][e]);
                mx = Tm::max_(mx, red);
                sum = W > 1 && single >= 0 ? exp2_((x1 - mx) * ct) : 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i * TEAM + i0 < nv) {
                        float add = 0.f;
#pragma unroll
                        for (int e = 0; e < W; ++e) add += exp2_(((float)x[i][e] - mx) * ct);
                        sum += add;
                    }
                sum = Tm::sum_(sum, red);
            }
        }
        if (!(MODE & STATS_IN) && p.stats && i0 == 0) { p.stats[2 * m] = mx; p.stats[2 * m + 1] = sum; }
        if ((MODE & LOSS) && threadIdx.x % TEAM < 64) {
            float kl = group_sum<64>(t.at >= 0 ? kl_part(t.p, st, mx, log2_(sum), p.temperature * (0.25f * LN2)) : 0.f);
            if (t.bad) kl = __builtin_nanf("");
            out = counts ? (double)w * kl : 0.0;
        }
        if (MODE & GRAD) {
            TG* d = (TG*)p.dlogits + m * p.ld_d;
            if (!counts) {
                if (!p.accumulate) for (int v = i0; v < V; v += TEAM) d[v] = (TG)0.f;
            } else {
                const float f = row_factor(p, scale, w, t.bad), fq = f * __builtin_amdgcn_rcpf(sum);
                const bool mine = threadIdx.x % TEAM < 64 && t.at >= 0;
                const float old = mine && p.accumulate ? (float)d[t.at] : 0.f;
                if (p.accumulate) Tm::sync();                // (the listed classes are read before anyone adds to them)
                VG* dv = reinterpret_cast<VG*>(d + head);
                auto put = [&](int i, const VS& y) {
                    VG o;
                    if (p.accumulate) o = dv[i];
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const float g = fq * exp2_(((float)y[e] - mx) * ct);
                        o[e] = (TG)(p.accumulate ? (float)o[e] + g : g);
                    }
                    dv[i] = o;
                };
                if (STREAM) walk<TEAM>(sv, i0, nv, put);
                else {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (i * TEAM + i0 < nv) put(i * TEAM + i0, x[i]);
                }
                if (W > 1 && single >= 0) {
                    const float g = fq * exp2_((x1 - mx) * ct);
                    d[single] = (TG)(p.accumulate ? (float)d[single] + g : g);
                }
                Tm::sync();                                  // the listed classes are written last
                if (mine) d[t.at] = (TG)(old + (fq * exp2_((st - mx) * ct) - f * t.p));
            }
        }
    }
    if (MODE & LOSS) {
        if (TEAM == 64) {
            if (lane == 0) parts[threadIdx.x >> 6] = out;
            __syncthreads();
            out = (parts[0] + parts[1]) + (parts[2] + parts[3]);
        }
        hand_over<BLOCK>(p, out, factor, parts);
    }
}

// loss = factor * (part[0] + part[1] + ...), in a fixed order
__global__ __launch_bounds__(1024) void distill_sum_kernel(const double* __restrict__ part, int n, double factor, float* __restrict__ loss) {
    __shared__ double red[16];
    double s = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < 16; ++w) t += red[w];
        *loss = (float)(t * factor);
    }
}

// ---------------------------------------------------------------- host
// Up to 512 classes: as few lanes a row (4 to 64) as hold its list and, 16 classes a lane, its logits: a wave's instructions then serve the
// most rows (131,072 x 300 bf16, 30 listed: loss 52 us with 16 classes a lane, 80 us with 8; 131,072 x 40 fp32: 13.0 and 13.9 us).
int lanes_of(int V, int k) {
    const int need = k > (V + 15) / 16 ? k : (V + 15) / 16;
    int g = 4;
    while (g < need) g *= 2;
    return g;
}
// workgroups of a launch over rows of up to 512 classes, and the rounds of each
int short_rounds(int M, int rows) { return (int)((((long)M + rows - 1) / rows + 2047) / 2048); }
int short_blocks(int M, int rows) {
    const long teams = ((long)M + rows - 1) / rows, rounds = short_rounds(M, rows);
    return (int)((teams + rounds - 1) / rounds);
}

int distill_check(const stes_distill_args* a, bool bwd) {
    STES_CHECK(a, STES_ERR_ARG, "stes_distill: null pointer");
    STES_CHECK(a->M >= 0 && a->V >= 1 && a->k >= 1, STES_ERR_ARG, "stes_distill: M >= 0, V >= 1 and k >= 1");
    STES_CHECK(a->k <= STES_DISTILL_MAX_K, STES_ERR_UNSUPPORTED, "stes_distill: at most 64 teacher classes a row");
    STES_CHECK(a->temperature >= 1e-6f && a->temperature <= 1e6f, STES_ERR_ARG, "stes_distill: the temperature lies between 1e-6 and 1e6");
    STES_CHECK(a->denom > 0.0, STES_ERR_ARG, "stes_distill: the denominator is positive");
    STES_CHECK(bwd || a->loss, STES_ERR_ARG, "stes_distill: loss is needed");
    if (!a->M) return STES_OK;
    STES_CHECK(a->V < 0x7fff0000, STES_ERR_UNSUPPORTED, "stes_distill: too many classes");
    STES_CHECK(a->V <= 8 * 64 || a->M < (1 << 22), STES_ERR_UNSUPPORTED, "stes_distill: more rows than a launch holds (2^32 threads)");
    STES_CHECK(a->logits && a->idx && a->val, STES_ERR_ARG, "stes_distill: null pointer");
    STES_CHECK(a->ld >= a->V && a->ld_idx >= a->k && a->ld_val >= a->k, STES_ERR_ARG, "stes_distill: rows overlap");
    STES_CHECK(!a->dlogits || a->ld_d >= a->V, STES_ERR_ARG, "stes_distill: rows of dlogits overlap");
    STES_CHECK(!bwd || (a->stats && a->dlogits), STES_ERR_ARG, "stes_distill_bwd: stats and dlogits are needed");
    STES_CHECK((uintptr_t)a->zeros % 8 == 0, STES_ERR_ARG, "stes_distill: zeros is aligned to 8 bytes");
    const int64_t need = bwd ? 0 : stes_distill_ws_floats(a->M, a->V, a->k, a->zeros != nullptr);
    STES_CHECK(!need || (a->ws && a->ws_floats >= need && (uintptr_t)a->ws % 8 == 0), STES_ERR_ARG, "stes_distill: workspace too small or not aligned to 8 bytes");
    const int64_t M = a->M;
    const StesRows stats = stes_flat(a->stats, 4, 2 * M), none{};
    const StesRows outs[5] = {{a->dlogits, a->d_f32 ? 4 : 2, a->ld_d, 0, M, 1, a->V}, stes_flat(bwd ? nullptr : a->loss, 4, 1), bwd ? none : stats, stes_flat(a->ws, 4, need),
                              stes_flat(bwd || M == 1 ? nullptr : a->zeros, 4, 2 * STES_DISTILL_WORDS)};
    const StesRows ins[6] = {{a->logits, a->f32 ? 4 : 2, a->ld, 0, M, 1, a->V}, {a->idx, a->idx_i64 ? 8 : 4, a->ld_idx, 0, M, 1, a->k}, {a->val, a->val_f32 ? 4 : 2, a->ld_val, 0, M, 1, a->k},
                             stes_flat(a->weight, 4, M), stes_flat(a->upstream, 4, 1), bwd ? stats : none};
    STES_CHECK(!stes_any_shared(outs, ins), STES_ERR_ARG, "stes_distill: what a call writes shares memory with what else it writes or reads");
    return STES_OK;
}

double loss_factor(const stes_distill_args& a) { return 4.0 * a.temperature / a.denom; }          // (the rows' parts are KL tau / 4)
float grad_factor(const stes_distill_args& a) { return (float)((double)a.grad_scale * a.temperature / a.denom); }

template <typename TS, typename TG, int G, int E, int MODE>
int launch_short(const stes_distill_args& a, hipStream_t s) {
    const int blocks = short_blocks(a.M, 256 / G);
    hipLaunchKernelGGL((distill_short_kernel<TS, TG, G, E, 256, MODE>), dim3(blocks), dim3(256), 0, s, a, short_rounds(a.M, 256 / G), loss_factor(a), grad_factor(a));
    return in_one_launch(a, blocks, 256) ? 0 : blocks;
}

template <typename TS, typename TG, int G, int MODE>
int launch_group(const stes_distill_args& a, hipStream_t s) {
    return a.V <= 8 * G ? launch_short<TS, TG, G, 8, MODE>(a, s) : launch_short<TS, TG, G, 16, MODE>(a, s);
}

template <typename TS, typename TG, int W, int TEAM, int N, bool STREAM, int MODE>
int launch_row(const stes_distill_args& a, hipStream_t s) {
    constexpr int RPB = TEAM == 64 ? 4 : 1;
    const int blocks = (int)(((long)a.M + RPB - 1) / RPB);
    hipLaunchKernelGGL((distill_row_kernel<TS, TG, W, TEAM, N, STREAM, MODE>), dim3(blocks), dim3(TEAM * RPB), 0, s, a, loss_factor(a), grad_factor(a));
    return in_one_launch(a, blocks, TEAM * RPB) ? 0 : blocks;
}

// -> how many partial sums the launch leaves in the workspace
template <typename TS, typename TG, int W, int MODE>
int launch_rows(const stes_distill_args& a, hipStream_t s) {
    if constexpr (W == 1) {
        return launch_row<TS, TG, 1, 256, 1, true, MODE>(a, s);
    } else {
        const int vecs = (a.V + W - 1) / W;
        if (vecs <= 64 * 8) return launch_row<TS, TG, W, 64, 8, false, MODE>(a, s);
        if (vecs <= 256 * 8) return launch_row<TS, TG, W, 256, 8, false, MODE>(a, s);
        if (vecs <= 512 * 8) return launch_row<TS, TG, W, 512, 8, false, MODE>(a, s);
        if (vecs <= 1024 * 8) return launch_row<TS, TG, W, 1024, 8, false, MODE>(a, s);
        if (vecs <= 1024 * 16 && (MODE & GRAD)) return launch_row<TS, TG, W, 1024, 16, false, MODE>(a, s);
        return launch_row<TS, TG, W, 1024, 1, true, MODE>(a, s);
    }
}

template <typename TS, typename TG, int MODE>
int launch_mode(const stes_distill_args& a, hipStream_t s) {
    if (a.V <= 8 * 64) {
        const int g = lanes_of(a.V, a.k);
        if (g == 4) return launch_group<TS, TG, 4, MODE>(a, s);
        if (g == 8) return launch_group<TS, TG, 8, MODE>(a, s);
        if (g == 16) return launch_group<TS, TG, 16, MODE>(a, s);
        if (g == 32) return launch_group<TS, TG, 32, MODE>(a, s);
        return launch_short<TS, TG, 64, 8, MODE>(a, s);
    }
    if constexpr (sizeof(TS) == sizeof(TG)) {
        // 16-byte accesses need the rows of logits and of dlogits at the same offset from a 16-byte boundary
        constexpr int W = 16 / sizeof(TS);
        const bool same = !(MODE & GRAD) || ((((uintptr_t)a.logits ^ (uintptr_t)a.dlogits) & 15) == 0 && (a.M == 1 || ((a.ld - a.ld_d) * (int)sizeof(TS) & 15) == 0));
        if (same && (uintptr_t)a.logits % sizeof(TS) == 0) return launch_rows<TS, TG, W, MODE>(a, s);
    }
    return launch_rows<TS, TG, 1, MODE>(a, s);
}

template <typename TS>
int launch(const stes_distill_args& a, bool bwd, hipStream_t s) {
    if (bwd) return a.d_f32 ? launch_mode<TS, float, GRAD | STATS_IN>(a, s) : launch_mode<TS, bf16, GRAD | STATS_IN>(a, s);
    if (!a.dlogits) return launch_mode<TS, TS, LOSS>(a, s);
    return a.d_f32 ? launch_mode<TS, float, LOSS | GRAD>(a, s) : launch_mode<TS, bf16, LOSS | GRAD>(a, s);
}

}  // namespace

extern "C" int64_t stes_distill_ws_floats(int M, int V, int k, int with_zeros) {
    if (M <= 1) return 0;
    const int blocks = V <= 8 * 64 ? short_blocks(M, 256 / lanes_of(V, k)) : M;          // (or fewer)
    return blocks == 1 || (with_zeros && blocks <= 16 * 256) ? 0 : 2 * (int64_t)blocks;          // (of 64 bits each)
}

extern "C" int stes_distill(const stes_distill_args* a, void* stream) {
    const int rc = distill_check(a, false);
    if (rc) return rc;
    int parts = 0;
    if (a->M) {
        parts = a->f32 ? launch<float>(*a, false, (hipStream_t)stream) : launch<bf16>(*a, false, (hipStream_t)stream);
        STES_LAUNCH_CHECK();
    }
    if (parts || !a->M) {                                    // (no rows: a sum of nothing)
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const double*)a->ws, parts, loss_factor(*a), a->loss);
        STES_LAUNCH_CHECK();
    }
    return STES_OK;
}

extern "C" int stes_distill_bwd(const stes_distill_args* a, void* stream) {
    const int rc = distill_check(a, true);
    if (rc) return rc;
    if (!a->M) return STES_OK;
    if (a->f32) launch<float>(*a, true, (hipStream_t)stream);
    else launch<bf16>(*a, true, (hipStream_t)stream);
    STES_LAUNCH_CHECK();
    return STES_OK;
}
