// Gated linear recurrence over sequences (stes_gated_scan_fwd / _bwd in include/stes.h).
//
// x_s = a_s x_{s-1} + z_s c_s with z = sigmoid(g), a = sigmoid(-g): an affine map of the state per step and channel.  Maps compose,
// (A, B) after (A', B') = (A A', A B' + B), so the time axis is cut: a thread takes L steps of V channels, a workgroup a block of
// STES_SCAN_BLOCK steps of a tile of channels, and the blocks of a sequence are joined while they run.  The backward pass is the
// same recurrence the other way round, k_{s-1} = a_s (dh_s + k_s), on states recomputed from the one in front of the block: it reads
// pre and dh and writes dpre, and stores no state but one per block.
//
// Joining the blocks of a sequence (T > STES_SCAN_BLOCK): workgroups draw tickets, all channels of a block of time before the
// next block, and a workgroup waits for lower tickets only, whose workgroups have started before it and wait for lower ones
// still: every wait ends.  Each block publishes its map (A, B) as soon as it has it and the state behind it when it knows the one in
// front; a later block walks back over published maps to the nearest published state.  Results do not depend on when words
// arrive.  Maps and states are single 64-bit words that are valid when they are not zero (A >= 0 carries its sign bit set, a state a
// one beside it), so relaxed atomics of agent scope carry them and no fence or cache write-back is needed.
//
// Bound: memory, one read of the inputs and one write of the outputs.  Measured (bf16, 768 channels, a copy of 1 GiB runs at 4,980 GB/s):
// one sequence of 65,536 frames forward 75 us (4.0 TB/s; 61 us without the joining, the rest is the walk back: 12 chains of 256
// blocks), 8 x 4,096 frames forward 41.5 us (3.6 TB/s) and backward 67 us (3.8 TB/s), 16 x 64 frames 5.4 and 7.5 us.
// (Comparisons here and below were made when the one sequence took 73 us: products that keep off 0 and gates that close cost the rest.)
// Why 256 steps x 64 channels (512 threads): halving the steps doubles the walk (86 us instead of 73 on the one long sequence); 128
// channels a row gain nothing over 64 (the lines of a row are whole either way); 32 would split them.  Why 4 steps a thread in bf16: with 8
// (tiles of 128 steps x 128 channels) a thread needs 197 registers forward and 256 backward: 86 us instead of 73 and 152 instead of 122.
#include "stes_common.h"

namespace {

// 16 bytes of a row, at any address that is a multiple of the element's size (global memory takes 16-byte accesses there)
template <typename T> struct Chunk;
template <> struct Chunk<bf16> { static constexpr int V = 8; typedef bf16x8 type; typedef bf16x8 anywhere __attribute__((aligned(2))); };
template <> struct Chunk<float> { static constexpr int V = 4; typedef f32x4 type; typedef f32x4 anywhere __attribute__((aligned(4))); };

// the first `left` elements of a chunk, the whole of it where left >= V
template <typename T>
__device__ __forceinline__ typename Chunk<T>::type load_chunk(const T* p, int left) {
    typename Chunk<T>::type r;
    if (left >= Chunk<T>::V) r = *reinterpret_cast<const typename Chunk<T>::anywhere*>(p);
    else {
#pragma unroll
        for (int v = 0; v < Chunk<T>::V; ++v) r[v] = v < left ? p[v] : (T)0.f;
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, typename Chunk<T>::type x, int left) {
    if (left >= Chunk<T>::V) *reinterpret_cast<typename Chunk<T>::anywhere*>(p) = x;
    else {
#pragma unroll
        for (int v = 0; v < Chunk<T>::V; ++v)
            if (v < left) p[v] = x[v];
    }
}

// The least fp32 number.  Added to products that could vanish (and lost in the rounding of all that are normal numbers), it keeps a product
// of a's above 0: infinity times it stays infinite, as it does step by step, and the largest finite state times it is 5e-7.
constexpr float LEAST = 0x1p-149f;
__device__ __forceinline__ float product(float a, float b) { return __builtin_fmaf(a, b, LEAST); }

// z = sigmoid(x) and a = sigmoid(-x), both to full relative precision (1 - z would lose a's digits where the gate is open).  A gate below -87
// closes: z goes to 0 with exp2's overflow (the lowest value of a type as a frame's mask, in its candidate too, adds nothing), and a is 1 there.
__device__ __forceinline__ void gate_pair(float x, float& z, float& a) {
    const float m = x * -1.4426950408889634f, e = __builtin_amdgcn_exp2f(m) + LEAST;
    z = __builtin_amdgcn_rcpf(1.f + e);
    a = m > 125.f ? 1.f : e * z;
}

__device__ __forceinline__ int seq_len(const stes_gated_scan_args& p, int b) {
    if (!p.lengths) return p.T;
    const int n = p.lengths[b];
    return n < 0 ? 0 : (n > p.T ? p.T : n);
}

// What another lane of this wave wrote to LDS is read next (a wave's LDS accesses are executed in order; this keeps the compiler's).
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---------------------------------------------------------------- joining blocks
struct Link { uint64_t* map; uint64_t* state; };     // [block][chain * CT + channel]

__device__ __forceinline__ void publish(uint64_t* w, uint64_t v) { __hip_atomic_store(w, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t peek(const uint64_t* w) { return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t map_word(float A, float B) { return ((uint64_t)__float_as_uint(B) << 32) | (__float_as_uint(A) | 0x80000000u); }
__device__ __forceinline__ uint64_t state_word(float x) { return ((uint64_t)__float_as_uint(x) << 32) | 1u; }

// a state through a block's map: one operation everywhere, so that it rounds alike everywhere
__device__ __forceinline__ float through(float A, float B, float x) { return __builtin_fmaf(A, x, B); }

constexpr int LOOK = 4;                  // blocks looked at in one round trip to memory (8: the polling itself costs 12 us of 73)
constexpr int REACH = 32;                // maps that a walk keeps; with so many it waits for the state behind them (16: 24 us instead of
                                         // 20 for 60,000 frames of 64 channels, one chain)
constexpr int MAX_ROUNDS = 1 << 22;      // (an exit for a broken workspace: the state becomes NaN)

// The state in front of block `blk` >= 1 of a channel (lane = channel): a walk back to the nearest published state, then that state
// through the maps of the blocks between, in their order.  Every state is its block's map of the state in front, so that is the same
// sequence of operations, and the same bits, wherever the walk ends.  `at` is the channel's word in a row of `words` words.
__device__ __forceinline__ float look_back(const Link& l, uint64_t (*kept)[64], long at, long words, int blk) {
    const int lane = threadIdx.x & 63;
    int depth = 0;                       // maps kept, of the blocks blk - 1, blk - 2, ...
    for (int round = 0; round < MAX_ROUNDS; ++round) {
        uint64_t st[LOOK], mp[LOOK];
#pragma unroll
        for (int k = 0; k < LOOK; ++k) {
            const int q = blk - 1 - depth - k < 0 ? 0 : blk - 1 - depth - k;
            st[k] = peek(l.state + q * words + at);
            mp[k] = peek(l.map + q * words + at);
        }
        const int before = depth;
        bool open = true, found = false;
        float x = 0.f;
#pragma unroll
        for (int k = 0; k < LOOK; ++k) {
            if (!open || blk - 1 - before - k < 0) continue;
            if (st[k]) { x = __uint_as_float((uint32_t)(st[k] >> 32)); found = true; open = false; }
            else if (mp[k] && depth < REACH) kept[depth++][lane] = mp[k];          // (block 0 publishes a state and no map)
            else open = false;
        }
        if (found) {
            for (int d = depth - 1; d >= 0; --d) {
                const uint64_t m = kept[d][lane];
                x = through(__uint_as_float((uint32_t)m & 0x7fffffffu), __uint_as_float((uint32_t)(m >> 32)), x);
            }
            return x;
        }
        if (depth == before) __builtin_amdgcn_s_sleep(1);
    }
    return __builtin_nanf("");
}

__global__ __launch_bounds__(256) void scan_clear_kernel(u32x4* __restrict__ w, long n) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) w[i] = (u32x4){0u, 0u, 0u, 0u};
}

// ---------------------------------------------------------------- tiles
// A workgroup of NT threads: LPR lanes side by side take 64 channels of a frame (128 bytes of bf16, 256 of fp32), NT / LPR segments
// of L steps one after the other in time.
template <typename T_, int LPR_, int L_>
struct Tile {
    typedef T_ T;
    static constexpr int V = Chunk<T>::V, LPR = LPR_, L = L_, CT = LPR * V, NS = STES_SCAN_BLOCK / L, NT = NS * LPR, NW = NT / 64, SW = 64 / LPR;
    static_assert(CT == 64, "a lane of a wave per channel");
};

struct Place { int b, c0, n, blk; long chain; };

template <class G, bool JOIN>
__device__ __forceinline__ Place place(const stes_gated_scan_args& p, int tiles, long chains, unsigned* ticket, unsigned* shared_ticket) {
    long id = blockIdx.x;
    Place r;
    r.blk = 0;
    if (JOIN) {
        if (threadIdx.x == 0) *shared_ticket = atomicAdd(ticket, 1u);
        __syncthreads();
        id = *shared_ticket;
        r.blk = (int)(id / chains);
    }
    r.chain = id - r.blk * chains;
    r.b = (int)(r.chain / tiles);
    r.c0 = (int)(r.chain - (long)r.b * tiles) * G::CT;
    r.n = seq_len(p, r.b);
    return r;
}

// A workgroup's share of the memory that the launch leaves zero, written by all but its first wave.
template <class G>
__device__ __forceinline__ void scrub(const stes_gated_scan_args& p) {
    u32x4* w = (u32x4*)p.scrub;
    constexpr int N = G::NT - 64;
    for (long i = (long)blockIdx.x * N + threadIdx.x - 64; i < p.scrub_bytes / 16; i += (long)gridDim.x * N) w[i] = (u32x4){0u, 0u, 0u, 0u};
}

template <class G, bool JOIN>
__global__ __launch_bounds__(G::NT) void scan_fwd_kernel(const stes_gated_scan_args p, int tiles, long chains, int blocks, unsigned* ticket, Link link) {
    typedef typename G::T T;
    typedef typename Chunk<T>::type VT;
    constexpr int V = G::V, L = G::L, CT = G::CT, SW = G::SW, NW = G::NW;
    __shared__ float sA[G::NS][CT], sB[G::NS][CT];       // maps of the segments, then of what precedes them in their wave
    __shared__ float tA[NW][CT], tB[NW][CT];             // maps of the waves; tB then: the state in front of each
    __shared__ uint64_t kept[JOIN ? REACH : 1][64];
    __shared__ unsigned drawn;
    const Place at = place<G, JOIN>(p, tiles, chains, ticket, &drawn);
    const int tid = threadIdx.x, cl = tid % G::LPR, seg = tid / G::LPR, lane = tid & 63, wave = tid >> 6;
    const int c = at.c0 + cl * V, n = at.n, s0 = at.blk * STES_SCAN_BLOCK + seg * L;
    const int left = p.H - c;
    const bool on = left > 0;
    const long H = p.H, step = p.reverse ? -p.ld_pre : p.ld_pre;
    const T* row = (const T*)p.pre + at.b * p.bs_pre + c + (p.reverse ? (long)(n - 1 - s0) : (long)s0) * p.ld_pre;
    VT g[L], cand[L];
#pragma unroll
    for (int j = 0; j < L; ++j)
        if (on && s0 + j < n) {
            g[j] = load_chunk<T>(row + j * step, left);
            cand[j] = load_chunk<T>(row + j * step + H, left);
        }
    float a[L][V], u[L][V], A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
    for (int j = 0; j < L; ++j) {
        if (on && s0 + j < n) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float z;
                gate_pair((float)g[j][v], z, a[j][v]);
                u[j][v] = z * (float)cand[j][v];
                A[v] *= a[j][v];
                B[v] = a[j][v] * B[v] + u[j][v];
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) { a[j][v] = 1.f; u[j][v] = 0.f; }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) { sA[seg][cl * V + v] = A[v] + LEAST; sB[seg][cl * V + v] = B[v]; }        // (product() above: 130 registers, one workgroup a CU)
    wave_lds_fence();
    {
        float fa = 1.f, fb = 0.f;                            // lane = channel
#pragma unroll
        for (int i = 0; i < SW; ++i) {
            const float ia = sA[wave * SW + i][lane], ib = sB[wave * SW + i][lane];
            sA[wave * SW + i][lane] = fa;
            sB[wave * SW + i][lane] = fb;
            fb = ia * fb + ib;
            fa = product(ia, fa);
        }
        tA[wave][lane] = fa;
        tB[wave][lane] = fb;
    }
    __syncthreads();
    if (JOIN && wave != 0 && p.scrub) scrub<G>(p);           // (while the first wave looks back)
    if (wave == 0) {
        const int ch = at.c0 + lane;
        float x = 0.f, fa[NW], fb[NW], mA = 1.f, mB = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) { fa[w] = tA[w][lane]; fb[w] = tB[w][lane]; mB = fa[w] * mB + fb[w]; mA = product(fa[w], mA); }
        const long word = at.chain * CT + lane, words = chains * CT;
        if (ch < p.H) {
            if (!JOIN || at.blk == 0) x = p.h0 ? p.h0[at.b * p.bs_h0 + ch] : 0.f;
            else {
                if (at.blk + 1 < blocks) publish(link.map + at.blk * words + word, map_word(mA, mB));
                x = look_back(link, kept, word, words, at.blk);
            }
            const float end = through(mA, mB, x);
            if (JOIN && at.blk + 1 < blocks) publish(link.state + at.blk * words + word, state_word(end));
            if (at.blk + 1 == blocks && p.h_last) p.h_last[at.b * p.bs_hl + ch] = end;
            if (p.states) p.states[((long)at.b * blocks + at.blk) * H + ch] = x;
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) { tB[w][lane] = x; x = fa[w] * x + fb[w]; }
    }
    __syncthreads();
    if (!on) return;
    float x[V];
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = sA[seg][cl * V + v] * tB[wave][cl * V + v] + sB[seg][cl * V + v];
    T* out = (T*)p.h + at.b * p.bs_h + c;
#pragma unroll
    for (int j = 0; j < L; ++j) {
        const int s = s0 + j;
        VT o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = a[j][v] * x[v] + u[j][v];
            o[v] = (T)(s < n ? x[v] : 0.f);
        }
        if (s < p.T) store_chunk<T>(out + (long)(p.reverse && s < n ? n - 1 - s : s) * p.ld_h, o, left);
    }
}

// blocks are drawn from the end of the sequence: block `at.blk` of the joining order is block blocks - 1 - at.blk of time
template <class G, bool JOIN>
__global__ __launch_bounds__(G::NT) void scan_bwd_kernel(const stes_gated_scan_args p, int tiles, long chains, int blocks, unsigned* ticket, Link link) {
    typedef typename G::T T;
    typedef typename Chunk<T>::type VT;
    constexpr int V = G::V, L = G::L, CT = G::CT, SW = G::SW, NW = G::NW;
    __shared__ float sA[G::NS][CT], sB[G::NS][CT], sR[G::NS][CT], sS[G::NS][CT];
    __shared__ float tA[NW][CT], tB[NW][CT], tR[NW][CT];             // tB and tR then: what comes to a wave from either side
    __shared__ uint64_t kept[JOIN ? REACH : 1][64];
    __shared__ unsigned drawn;
    const Place at = place<G, JOIN>(p, tiles, chains, ticket, &drawn);
    const int blk = blocks - 1 - at.blk;
    const int tid = threadIdx.x, cl = tid % G::LPR, seg = tid / G::LPR, lane = tid & 63, wave = tid >> 6;
    const int c = at.c0 + cl * V, n = at.n, s0 = blk * STES_SCAN_BLOCK + seg * L;
    const int left = p.H - c;
    const bool on = left > 0;
    const long H = p.H, t0 = p.reverse ? (long)(n - 1 - s0) : (long)s0, sign = p.reverse ? -1 : 1;
    const T* row = (const T*)p.pre + at.b * p.bs_pre + c + t0 * p.ld_pre;
    const T* drow = p.dh ? (const T*)p.dh + at.b * p.bs_dh + c + t0 * p.ld_dh : nullptr;
    VT g[L], cand[L], d[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
        const bool live = on && s0 + j < n;
#pragma unroll
        for (int v = 0; v < V; ++v) d[j][v] = (T)0.f;
        if (live) {
            g[j] = load_chunk<T>(row + sign * j * p.ld_pre, left);
            cand[j] = load_chunk<T>(row + sign * j * p.ld_pre + H, left);
            if (drow) d[j] = load_chunk<T>(drow + sign * j * p.ld_dh, left);
        }
    }
    // the segment's maps, forwards (A, B) and backwards (A, R)
    float A[V], B[V], R[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; R[v] = 0.f; }
#pragma unroll
    for (int j = 0; j < L; ++j) {
        // (selects, not a branch: the gates then stay in registers for the passes below; recomputed, 60 % more time on short sequences)
        const bool live = on && s0 + j < n;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float z, k;
            gate_pair((float)g[j][v], z, k);
            k = live ? k : 1.f;
            const float u = live ? z * (float)cand[j][v] : 0.f;
            B[v] = k * B[v] + u;
            A[v] = product(A[v], k);
            R[v] += A[v] * (float)d[j][v];               // d_j reaches the segment's front through a_0 .. a_j
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) { sA[seg][cl * V + v] = A[v]; sB[seg][cl * V + v] = B[v]; sR[seg][cl * V + v] = R[v]; }
    wave_lds_fence();
    {
        float ia[SW], ib[SW], ir[SW], fa = 1.f, fb = 0.f, ra = 1.f, rr = 0.f;          // lane = channel
#pragma unroll
        for (int i = 0; i < SW; ++i) { ia[i] = sA[wave * SW + i][lane]; ib[i] = sB[wave * SW + i][lane]; ir[i] = sR[wave * SW + i][lane]; }
#pragma unroll
        for (int i = 0; i < SW; ++i) {
            sA[wave * SW + i][lane] = fa;
            sB[wave * SW + i][lane] = fb;
            fb = ia[i] * fb + ib[i];
            fa = product(ia[i], fa);
        }
#pragma unroll
        for (int i = SW - 1; i >= 0; --i) {
            sS[wave * SW + i][lane] = ra;
            sR[wave * SW + i][lane] = rr;
            rr = ia[i] * rr + ir[i];
            ra = product(ia[i], ra);
        }
        tA[wave][lane] = fa;
        tB[wave][lane] = fb;
        tR[wave][lane] = rr;
    }
    __syncthreads();
    if (JOIN && wave != 0 && p.scrub) scrub<G>(p);
    if (wave == 0) {
        const int ch = at.c0 + lane;
        float fa[NW], fb[NW], fr[NW], mA = 1.f, mR = 0.f, x = 0.f, k = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) { fa[w] = tA[w][lane]; fb[w] = tB[w][lane]; fr[w] = tR[w][lane]; }
#pragma unroll
        for (int w = NW - 1; w >= 0; --w) { mR = fa[w] * mR + fr[w]; mA = product(fa[w], mA); }
        const long word = at.chain * CT + lane, words = chains * CT;
        if (ch < p.H) {
            x = p.states[((long)at.b * blocks + blk) * H + ch];
            if (!JOIN || at.blk == 0) k = p.dh_last ? p.dh_last[at.b * p.bs_dhl + ch] : 0.f;
            else {
                if (blk) publish(link.map + at.blk * words + word, map_word(mA, mR));
                k = look_back(link, kept, word, words, at.blk);
            }
            const float front = through(mA, mR, k);
            if (JOIN && blk) publish(link.state + at.blk * words + word, state_word(front));
            if (!blk && p.dh0) p.dh0[at.b * H + ch] = front;
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) { tB[w][lane] = x; x = fa[w] * x + fb[w]; }
#pragma unroll
        for (int w = NW - 1; w >= 0; --w) { tR[w][lane] = k; k = fa[w] * k + fr[w]; }
    }
    __syncthreads();
    if (!on) return;
    float x[L][V], k[V];                                     // the state in front of each step; what comes from the steps behind
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int q = cl * V + v;
        x[0][v] = sA[seg][q] * tB[wave][q] + sB[seg][q];
        k[v] = sS[seg][q] * tR[wave][q] + sR[seg][q];
    }
#pragma unroll
    for (int j = 0; j + 1 < L; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float z, w;
            gate_pair((float)g[j][v], z, w);
            x[j + 1][v] = s0 + j < n ? w * x[j][v] + z * (float)cand[j][v] : 0.f;
        }
    T* out = (T*)p.dpre + at.b * p.bs_dpre + c;
#pragma unroll
    for (int j = L - 1; j >= 0; --j) {
        const int s = s0 + j;
        if (s >= p.T) continue;
        VT og, oc;
        if (s < n) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float z, w;
                gate_pair((float)g[j][v], z, w);
                const float lam = (float)d[j][v] + k[v];
                oc[v] = (T)(lam * z);
                og[v] = (T)(lam * z * ((float)cand[j][v] - x[j][v]) * w);       // (in this order: the difference may be of the type's lowest value, z then 0)
                k[v] = w * lam;
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) og[v] = oc[v] = (T)0.f;
        }
        T* o = out + (long)(p.reverse && s < n ? n - 1 - s : s) * p.ld_dpre;
        store_chunk<T>(o, og, left);
        store_chunk<T>(o + H, oc, left);
    }
}

// ---------------------------------------------------------------- few steps
// T <= SHORT: a thread walks all steps of V channels; nothing is shared (frames of streams, one at a time: 3.8 us for one stream of 768
// channels, 5 us for 192, where a tile would have 1 of its 64 segments at work).  All loads are issued before the first step.
constexpr int SHORT = 8;

template <typename T, bool BWD>
__global__ __launch_bounds__(64) void scan_short_kernel(const stes_gated_scan_args p, long groups) {
    typedef typename Chunk<T>::type VT;
    constexpr int V = Chunk<T>::V;
    const long id = (long)blockIdx.x * 64 + threadIdx.x, per = (p.H + V - 1) / V;
    if (id >= groups) return;
    const int b = (int)(id / per), c = (int)(id - b * per) * V, n = seq_len(p, b), left = p.H - c;
    const long H = p.H;
    const T* pre = (const T*)p.pre + b * p.bs_pre + c;
    const T* dh = BWD && p.dh ? (const T*)p.dh + b * p.bs_dh + c : nullptr;
    VT g[SHORT], cand[SHORT], d[BWD ? SHORT : 1];
#pragma unroll
    for (int s = 0; s < SHORT; ++s)
        if (s < n) {
            const long t = p.reverse ? n - 1 - s : s;
            g[s] = load_chunk<T>(pre + t * p.ld_pre, left);
            cand[s] = load_chunk<T>(pre + t * p.ld_pre + H, left);
            if (BWD && dh) d[s] = load_chunk<T>(dh + t * p.ld_dh, left);
        }
    float x[V], before[BWD ? SHORT : 1][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        x[v] = 0.f;
        if (v >= left) continue;
        if (BWD) { if (p.T) x[v] = p.states[b * H + c + v]; }
        else {
            if (p.h0) x[v] = p.h0[b * p.bs_h0 + c + v];
            if (p.states && p.T) p.states[b * H + c + v] = x[v];
        }
    }
#pragma unroll
    for (int s = 0; s < SHORT; ++s) {
        if (s >= p.T) break;
        VT o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (BWD) before[s][v] = x[v];
            if (s < n) {
                float z, a;
                gate_pair((float)g[s][v], z, a);
                x[v] = a * x[v] + z * (float)cand[s][v];
            }
            o[v] = (T)(s < n ? x[v] : 0.f);
        }
        if (!BWD) store_chunk<T>((T*)p.h + b * p.bs_h + c + (long)(p.reverse && s < n ? n - 1 - s : s) * p.ld_h, o, left);
    }
    if (!BWD) {
        if (p.h_last)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < left) p.h_last[b * p.bs_hl + c + v] = x[v];
        return;
    }
    float k[V];
#pragma unroll
    for (int v = 0; v < V; ++v) k[v] = p.dh_last && v < left ? p.dh_last[b * p.bs_dhl + c + v] : 0.f;
#pragma unroll
    for (int s = SHORT - 1; s >= 0; --s) {
        if (s >= p.T) continue;
        VT og, oc;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            og[v] = oc[v] = (T)0.f;
            if (s < n) {
                float z, a;
                gate_pair((float)g[s][v], z, a);
                const float lam = (dh ? (float)d[BWD ? s : 0][v] : 0.f) + k[v];
                oc[v] = (T)(lam * z);
                og[v] = (T)(lam * z * ((float)cand[s][v] - before[BWD ? s : 0][v]) * a);
                k[v] = a * lam;
            }
        }
        T* o = (T*)p.dpre + b * p.bs_dpre + c + (long)(p.reverse && s < n ? n - 1 - s : s) * p.ld_dpre;
        store_chunk<T>(o, og, left);
        store_chunk<T>(o + H, oc, left);
    }
    if (p.dh0)
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < left) p.dh0[b * H + c + v] = k[v];
}

// The gradient of an initial state that the batch shares: 16 strands of rows per channel, each added up in order, then the strands.
__global__ __launch_bounds__(1024) void scan_dh0_sum_kernel(const float* __restrict__ dh0, float* __restrict__ out, int B, int H) {
    __shared__ float part[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), strand = threadIdx.x >> 6;
    float s = 0.f;
    if (c < H) {
#pragma unroll 4
        for (int b = strand; b < B; b += 16) s += dh0[(long)b * H + c];
    }
    part[strand][threadIdx.x & 63] = s;
    __syncthreads();
    if (strand || c >= H) return;
    for (int k = 1; k < 16; ++k) s += part[k][threadIdx.x];
    out[c] = s;
}

// ---------------------------------------------------------------- host
constexpr int CT = 64;                       // channels of a tile, of either type

int blocks_of(int T) { return T / STES_SCAN_BLOCK + (T % STES_SCAN_BLOCK != 0); }
// words of one kind in the workspace
long words_of(int B, int T, int H) { return (long)blocks_of(T) * B * ((H + CT - 1) / CT * CT); }

// rows of `width` elements that a call writes: frames within sequences or the reverse, apart from one another
bool apart(int64_t ld, int T, int64_t bs, int B, int64_t width) {
    if (B <= 1) return T <= 1 || ld >= width;
    if (T <= 1) return bs >= width;
    return ld <= bs ? ld >= width && bs >= ld * (T - 1) + width : bs >= width && ld >= bs * (B - 1) + width;
}

int scan_check(const stes_gated_scan_args* a, bool bwd) {
    STES_CHECK(a, STES_ERR_ARG, "stes_gated_scan: null pointer");
    STES_CHECK(a->B >= 0 && a->T >= 0 && a->H >= 0, STES_ERR_ARG, "stes_gated_scan: negative size");
    STES_CHECK(a->f32 == 0 || a->f32 == 1, STES_ERR_ARG, "stes_gated_scan: f32 is 0 (bf16) or 1 (fp32)");
    STES_CHECK(!a->dh0_sum || a->dh0 || !a->B, STES_ERR_ARG, "stes_gated_scan_bwd: dh0_sum needs dh0");
    if (!a->B || !a->H) return STES_OK;
    STES_CHECK(a->H <= (1 << 24) && a->B <= (1 << 24) && (long)a->B * ((a->H + CT - 1) / CT) * (blocks_of(a->T) + 1) < (1L << 23), STES_ERR_UNSUPPORTED,
               "stes_gated_scan: more tiles than a launch holds (2^32 threads)");
    if (a->T) {
        STES_CHECK(a->pre && a->ld_pre >= 2L * a->H && a->bs_pre >= 0, STES_ERR_ARG, "stes_gated_scan: pre is [B][T][2H]");
        if (!bwd) STES_CHECK(a->h && apart(a->ld_h, a->T, a->bs_h, a->B, a->H), STES_ERR_ARG, "stes_gated_scan_fwd: h is [B][T][H], rows apart");
        else {
            STES_CHECK(a->states && a->dpre, STES_ERR_ARG, "stes_gated_scan_bwd: states and dpre are needed");
            STES_CHECK(apart(a->ld_dpre, a->T, a->bs_dpre, a->B, 2L * a->H), STES_ERR_ARG, "stes_gated_scan_bwd: dpre is [B][T][2H], rows apart");
            STES_CHECK(!a->dh || (a->ld_dh >= a->H && a->bs_dh >= 0), STES_ERR_ARG, "stes_gated_scan_bwd: dh is [B][T][H]");
        }
        const int64_t need = stes_gated_scan_ws_bytes(a->B, a->T, a->H);
        STES_CHECK(need == 0 || (a->ws && a->ws_bytes >= need && (uintptr_t)a->ws % 16 == 0), STES_ERR_ARG, "stes_gated_scan: workspace too small or not aligned to 16 bytes");
    }
    STES_CHECK(!a->scrub || (a->T > STES_SCAN_BLOCK && a->scrub_bytes >= 0 && a->scrub_bytes % 16 == 0 && (uintptr_t)a->scrub % 16 == 0), STES_ERR_ARG,
               "stes_gated_scan: scrub goes with more than STES_SCAN_BLOCK steps, in multiples of 16 bytes");
    STES_CHECK(!a->h0 || a->bs_h0 == 0 || a->bs_h0 >= a->H, STES_ERR_ARG, "stes_gated_scan: rows of h0 overlap");
    STES_CHECK(!a->h_last || a->bs_hl >= a->H, STES_ERR_ARG, "stes_gated_scan: rows of h_last overlap");
    STES_CHECK(!(a->h_last && a->h_last == a->h0) || a->bs_h0 == a->bs_hl, STES_ERR_ARG, "stes_gated_scan: a state in place keeps its row stride");
    STES_CHECK(!bwd || !a->dh_last || a->bs_dhl == 0 || a->bs_dhl >= a->H, STES_ERR_ARG, "stes_gated_scan_bwd: rows of dh_last overlap");
    const int64_t T = a->T, B = a->B, H = a->H, one = B > 1;
    const int es = a->f32 ? 4 : 2;
    const StesRows pre{a->pre, es, a->ld_pre, a->bs_pre, T, B, 2 * H}, h{a->h, es, a->ld_h, a->bs_h, T, B, H}, len{a->lengths, 4, 0, 1, 1, B, 1},
        h0{a->h0, 4, 0, a->bs_h0, 1, a->bs_h0 ? B : 1, H}, last{a->h_last, 4, 0, a->bs_hl, 1, B, H}, states{a->states, 4, H, blocks_of(a->T) * H, blocks_of(a->T), B, H},
        dh{a->dh, es, a->ld_dh, a->bs_dh, T, B, H}, dlast{a->dh_last, 4, 0, a->bs_dhl, 1, a->bs_dhl ? B : 1, H},
        dpre{a->dpre, es, a->ld_dpre, a->bs_dpre, T, B, 2 * H}, dh0{a->dh0, 4, 0, H, 1, B, H}, total{a->dh0_sum, 4, 0, H, 1, 1, H};
    const StesRows none{};
    const StesRows outs[5] = {bwd ? dpre : h, bwd ? dh0 : last, bwd ? total : states, stes_flat(a->ws, 1, stes_gated_scan_ws_bytes(a->B, a->T, a->H)),
                              stes_flat(a->scrub, 1, a->scrub_bytes)}, ins[5] = {pre, len, bwd ? states : h0, bwd ? dh : none, bwd ? dlast : none};
    const bool in_place = !bwd && a->h_last == a->h0;                       // (checked above)
    STES_CHECK(!stes_any_shared(outs, ins, in_place ? 1 : -1, 2), STES_ERR_ARG, "stes_gated_scan: what a call writes shares memory with what else it writes or reads");
    return STES_OK;
}

template <class G, bool BWD>
void launch_tiles(const stes_gated_scan_args& a, hipStream_t s) {
    static_assert(G::CT == CT, "the workspace is laid out for tiles of CT channels");
    const int tiles = (a.H + G::CT - 1) / G::CT, blocks = blocks_of(a.T);
    const long chains = (long)a.B * tiles;
    unsigned* ticket = (unsigned*)a.ws;
    uint64_t* words = (uint64_t*)((char*)a.ws + 256);
    const Link link{words, words + words_of(a.B, a.T, a.H)};
    if (blocks > 1) {
        const long n = stes_gated_scan_ws_bytes(a.B, a.T, a.H) / 16;
        if (!a.ws_zero) hipLaunchKernelGGL(scan_clear_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, (u32x4*)a.ws, n);
        if (BWD) hipLaunchKernelGGL((scan_bwd_kernel<G, true>), dim3((unsigned)(chains * blocks)), dim3(G::NT), 0, s, a, tiles, chains, blocks, ticket, link);
        else hipLaunchKernelGGL((scan_fwd_kernel<G, true>), dim3((unsigned)(chains * blocks)), dim3(G::NT), 0, s, a, tiles, chains, blocks, ticket, link);
    } else {
        if (BWD) hipLaunchKernelGGL((scan_bwd_kernel<G, false>), dim3((unsigned)chains), dim3(G::NT), 0, s, a, tiles, chains, 1, ticket, link);
        else hipLaunchKernelGGL((scan_fwd_kernel<G, false>), dim3((unsigned)chains), dim3(G::NT), 0, s, a, tiles, chains, 1, ticket, link);
    }
}

template <typename T, bool BWD>
void scan_launch(const stes_gated_scan_args& a, hipStream_t s) {
    if (a.T <= SHORT) {
        const long groups = (long)a.B * ((a.H + Chunk<T>::V - 1) / Chunk<T>::V);
        hipLaunchKernelGGL((scan_short_kernel<T, BWD>), dim3((unsigned)((groups + 63) / 64)), dim3(64), 0, s, a, groups);
    } else if constexpr (sizeof(T) == 2) launch_tiles<Tile<T, 8, 4>, BWD>(a, s);
    else launch_tiles<Tile<T, 16, 8>, BWD>(a, s);
}

}  // namespace

extern "C" int64_t stes_gated_scan_ws_bytes(int B, int T, int H) {
    if (B <= 0 || H <= 0 || T <= STES_SCAN_BLOCK) return 0;
    return 256 + 16 * words_of(B, T, H);
}

extern "C" int stes_gated_scan_fwd(const stes_gated_scan_args* a, void* stream) {
    const int rc = scan_check(a, false);
    if (rc) return rc;
    if (!a->B || !a->H) return STES_OK;
    if (a->f32) scan_launch<float, false>(*a, (hipStream_t)stream);
    else scan_launch<bf16, false>(*a, (hipStream_t)stream);
    STES_LAUNCH_CHECK();
    return STES_OK;
}

extern "C" int stes_gated_scan_bwd(const stes_gated_scan_args* a, void* stream) {
    const int rc = scan_check(a, true);
    if (rc) return rc;
    if (!a->H) return STES_OK;
    if (a->B) {
        if (a->f32) scan_launch<float, true>(*a, (hipStream_t)stream);
        else scan_launch<bf16, true>(*a, (hipStream_t)stream);
        STES_LAUNCH_CHECK();
    }
    if (a->dh0_sum) {                                       // (zeros for an empty batch)
        hipLaunchKernelGGL(scan_dh0_sum_kernel, dim3((a->H + 63) / 64), dim3(1024), 0, (hipStream_t)stream, a->dh0, a->dh0_sum, a->B, a->H);
        STES_LAUNCH_CHECK();
    }
    return STES_OK;
}
