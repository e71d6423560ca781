// Distillation from a teacher's top logits (stes_distill / stes_distill_bwd in include/stes.h): the temperature-scaled KL divergence
// of the student's softmax over all V classes from the teacher's softmax over its k best, and its gradient.
#include "stes_common.h"

namespace {

struct Entry { int at; float p; };          // one listed class of a row: its index (-1: none) and its probability, duplicates merged

// The teacher's distribution of a row, one entry per lane of a wave (k <= 64).  -> bad: an index beyond V.  An index that is
// listed again keeps its whole probability at its first place; the later places hold at < 0.
__device__ __forceinline__ Entry teacher_row(const stes_distill_args& p, long m, int lane, bool& some, bool& bad) {
    Entry e{-1, 0.f};
    float v = -INFINITY;
    if (lane < p.k) {
        const long o = m * p.ld_idx + lane;
        const long i = p.idx_i64 ? ((const int64_t*)p.idx)[o] : (long)((const int32_t*)p.idx)[o];
        e.at = i < 0 ? -1 : (i >= p.V ? p.V : (int)i);
        const long ov = m * p.ld_val + lane;
        if (i >= 0) v = p.val_f32 ? ((const float*)p.val)[ov] : (float)((const bf16*)p.val)[ov];
    }
    bad = __any(e.at >= p.V);
    float mx = v;
    bool nan = v != v;
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    bad = bad || __any(nan) || mx == INFINITY;
    some = mx > -INFINITY || bad;
    e.p = v > -INFINITY ? __expf((v - mx) / p.temperature) : 0.f;
    e.p /= wave_sum(e.p);
    float whole = 0.f;
    bool first = true;
    for (int j = 0; j < p.k; ++j) {
        const int aj = __shfl(e.at, j, 64);
        const float pj = __shfl(e.p, j, 64);
        if (aj == e.at) { whole += pj; first = first && j >= lane; }
    }
    e.p = whole;
    if (!first) e.at = -1;
    return e;
}

__device__ __forceinline__ float block_max(float v, float* red) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = fmaxf(v, red[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v += red[w];
    return v;
}

template <typename TS, typename TG>
__global__ __launch_bounds__(256) void distill_row_kernel(const stes_distill_args p, int have_stats, int want_loss) {
    __shared__ float red[4];
    const long m = blockIdx.x;
    const TS* s = (const TS*)p.logits + m * p.ld;
    TG* d = p.dlogits ? (TG*)p.dlogits + m * p.ld_d : nullptr;
    const float w = p.weight ? p.weight[m] : 1.f, it = 1.f / p.temperature;
    const int lane = threadIdx.x & 63;
    bool some, bad;
    const Entry e = teacher_row(p, m, lane, some, bad);
    if (!some || w == 0.f) {
        if (want_loss && threadIdx.x == 0) p.ws[m] = 0.f;
        if (p.stats && !have_stats && threadIdx.x == 0) { p.stats[2 * m] = 0.f; p.stats[2 * m + 1] = 0.f; }
        if (d && !p.accumulate) for (int v = threadIdx.x; v < p.V; v += 256) d[v] = (TG)0.f;
        return;
    }
    float mx, inv;
    if (have_stats) { mx = p.stats[2 * m]; inv = p.stats[2 * m + 1]; }
    else {
        mx = -INFINITY;
        for (int v = threadIdx.x; v < p.V; v += 256) mx = fmaxf(mx, (float)s[v]);
        mx = block_max(mx, red);
        float sum = 0.f;
        for (int v = threadIdx.x; v < p.V; v += 256) sum += __expf(((float)s[v] - mx) * it);
        sum = block_sum(sum, red);
        inv = 1.f / sum;
        if (p.stats && threadIdx.x == 0) { p.stats[2 * m] = mx; p.stats[2 * m + 1] = inv; }
    }
    const float sv = e.at >= 0 && e.at < p.V ? (float)s[e.at] : 0.f;
    if (want_loss && threadIdx.x < 64) {
        float kl = e.at >= 0 && e.p > 0.f ? e.p * (logf(e.p) - ((sv - mx) * it + logf(inv))) : 0.f;
        kl = wave_sum(kl);
        if (bad) kl = NAN;
        if (threadIdx.x == 0) p.ws[m] = w * kl;
    }
    if (!d) return;
    float f = (float)((double)p.temperature / p.denom) * p.grad_scale * w * (p.upstream ? p.upstream[0] : 1.f);
    if (bad) f = NAN;
    // the listed classes are written last, by the lanes that hold them: read what they add to first
    const bool mine = threadIdx.x < 64 && e.at >= 0 && e.at < p.V && e.p > 0.f;
    const float old = mine && p.accumulate ? (float)d[e.at] : 0.f;
    __syncthreads();
    for (int v = threadIdx.x; v < p.V; v += 256) {
        const float g = f * (__expf(((float)s[v] - mx) * it) * inv);
        d[v] = (TG)(p.accumulate ? (float)d[v] + g : g);
    }
    __syncthreads();
    if (mine) d[e.at] = (TG)(old + f * (__expf((sv - mx) * it) * inv - e.p));
}

// loss = factor * (part[0] + part[1] + ...), in a fixed order
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ part, int n, double factor, float* __restrict__ loss) {
    __shared__ double red[16];
    double s = 0.0;
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

int distill_check(const stes_distill_args* a, bool bwd) {
    STES_CHECK(a, STES_ERR_ARG, "stes_distill: null pointer");
    STES_CHECK(a->M >= 0 && a->V >= 1 && a->k >= 1, STES_ERR_ARG, "stes_distill: M >= 0, V >= 1 and k >= 1");
    STES_CHECK(a->k <= STES_DISTILL_MAX_K, STES_ERR_UNSUPPORTED, "stes_distill: at most 64 teacher classes a row");
    STES_CHECK(a->temperature > 0.f && a->temperature < INFINITY, STES_ERR_ARG, "stes_distill: the temperature is positive");
    STES_CHECK(a->denom > 0.0, STES_ERR_ARG, "stes_distill: the denominator is positive");
    STES_CHECK(bwd || a->loss, STES_ERR_ARG, "stes_distill: loss is needed");
    if (!a->M) return STES_OK;
    STES_CHECK(a->logits && a->idx && a->val, STES_ERR_ARG, "stes_distill: null pointer");
    STES_CHECK(a->ld >= a->V && a->ld_idx >= a->k && a->ld_val >= a->k, STES_ERR_ARG, "stes_distill: rows overlap");
    STES_CHECK(!a->dlogits || a->ld_d >= a->V, STES_ERR_ARG, "stes_distill: rows of dlogits overlap");
    STES_CHECK(a->dlogits != a->logits, STES_ERR_ARG, "stes_distill: dlogits must not be logits");
    STES_CHECK(!bwd || (a->stats && a->dlogits), STES_ERR_ARG, "stes_distill_bwd: stats and dlogits are needed");
    STES_CHECK(bwd || (a->ws && a->ws_floats >= stes_distill_ws_floats(a->M, a->V)), STES_ERR_ARG, "stes_distill: workspace too small");
    return STES_OK;
}

template <typename TS>
void distill_launch(const stes_distill_args& a, bool bwd, hipStream_t s) {
    if (a.d_f32) hipLaunchKernelGGL((distill_row_kernel<TS, float>), dim3(a.M), dim3(256), 0, s, a, (int)bwd, (int)!bwd);
    else hipLaunchKernelGGL((distill_row_kernel<TS, bf16>), dim3(a.M), dim3(256), 0, s, a, (int)bwd, (int)!bwd);
}

}  // namespace

extern "C" int64_t stes_distill_ws_floats(int M, int V) {
    (void)V;
    return M > 0 ? M : 1;
}

extern "C" int stes_distill(const stes_distill_args* a, void* stream) {
    const int rc = distill_check(a, false);
    if (rc) return rc;
    if (a->M) {
        if (a->f32) distill_launch<float>(*a, false, (hipStream_t)stream);
        else distill_launch<bf16>(*a, false, (hipStream_t)stream);
        STES_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a->ws, a->M, (double)a->temperature * a->temperature / a->denom, a->loss);
    STES_LAUNCH_CHECK();
    return STES_OK;
}

extern "C" int stes_distill_bwd(const stes_distill_args* a, void* stream) {
    const int rc = distill_check(a, true);
    if (rc) return rc;
    if (!a->M) return STES_OK;
    if (a->f32) distill_launch<float>(*a, true, (hipStream_t)stream);
    else distill_launch<bf16>(*a, true, (hipStream_t)stream);
    STES_LAUNCH_CHECK();
    return STES_OK;
}
