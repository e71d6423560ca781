// Gated linear recurrence over sequences (stes_gated_scan_fwd / _bwd in include/stes.h).
//
// x_s = a_s x_{s-1} + z_s c_s with z = sigmoid(g), a = sigmoid(-g): an affine map of the state per step and channel, so runs of
// steps compose, (A, B) after (A', B') = (A A', A B' + B), and channels are independent.
#include "stes_common.h"

namespace {

// z = sigmoid(x) and a = sigmoid(-x), both to full relative precision (1 - z would lose a's digits where the gate is open)
__device__ __forceinline__ void gate_pair(float x, float& z, float& a) {
    const float t = __expf(-fabsf(x));
    const float big = __builtin_amdgcn_rcpf(1.f + t), small = t * big;
    z = x >= 0.f ? big : small;
    a = x >= 0.f ? small : big;
}

__device__ __forceinline__ int seq_len(const stes_gated_scan_args& p, int b) {
    if (!p.lengths) return p.T;
    const int n = p.lengths[b];
    return n < 0 ? 0 : (n > p.T ? p.T : n);
}

// One thread per (sequence, channel), step by step.
template <typename T>
__global__ __launch_bounds__(64) void scan_fwd_serial_kernel(const stes_gated_scan_args p) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= p.H) return;
    const int n = seq_len(p, b), nb = (p.T + STES_SCAN_BLOCK - 1) / STES_SCAN_BLOCK;
    const T* pre = (const T*)p.pre + (long)b * p.bs_pre + c;
    T* h = (T*)p.h + (long)b * p.bs_h + c;
    float x = p.h0 ? p.h0[(long)b * p.bs_h0 + c] : 0.f;
    for (int s = 0; s < p.T; ++s) {
        if (p.states && s % STES_SCAN_BLOCK == 0) p.states[((long)b * nb + s / STES_SCAN_BLOCK) * p.H + c] = x;
        if (s < n) {
            const int t = p.reverse ? n - 1 - s : s;
            float z, a;
            gate_pair((float)pre[t * p.ld_pre], z, a);
            x = a * x + z * (float)pre[t * p.ld_pre + p.H];
            h[t * p.ld_h] = (T)x;
        } else {
            h[s * p.ld_h] = (T)0.f;
        }
    }
    if (p.h_last) p.h_last[(long)b * p.bs_hl + c] = x;
}

template <typename T>
__global__ __launch_bounds__(64) void scan_bwd_serial_kernel(const stes_gated_scan_args p) {
    __shared__ float xs[STES_SCAN_BLOCK][64];
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= p.H) return;
    const int n = seq_len(p, b), nb = (p.T + STES_SCAN_BLOCK - 1) / STES_SCAN_BLOCK;
    const T* pre = (const T*)p.pre + (long)b * p.bs_pre + c;
    const T* dh = p.dh ? (const T*)p.dh + (long)b * p.bs_dh + c : nullptr;
    T* dpre = (T*)p.dpre + (long)b * p.bs_dpre + c;
    float carry = p.dh_last ? p.dh_last[(long)b * p.bs_dhl + c] : 0.f;
    for (int s = n; s < p.T; ++s) { dpre[s * p.ld_dpre] = (T)0.f; dpre[s * p.ld_dpre + p.H] = (T)0.f; }
    for (int blk = nb - 1; blk >= 0; --blk) {
        const int s0 = blk * STES_SCAN_BLOCK, s1 = min(n, s0 + STES_SCAN_BLOCK);
        float x = p.states[((long)b * nb + blk) * p.H + c];
        for (int s = s0; s < s1; ++s) {
            const int t = p.reverse ? n - 1 - s : s;
            float z, a;
            gate_pair((float)pre[t * p.ld_pre], z, a);
            xs[s - s0][threadIdx.x] = x;
            x = a * x + z * (float)pre[t * p.ld_pre + p.H];
        }
        for (int s = s1 - 1; s >= s0; --s) {
            const int t = p.reverse ? n - 1 - s : s;
            float z, a;
            gate_pair((float)pre[t * p.ld_pre], z, a);
            const float l = carry + (dh ? (float)dh[t * p.ld_dh] : 0.f);
            dpre[t * p.ld_dpre] = (T)(l * ((float)pre[t * p.ld_pre + p.H] - xs[s - s0][threadIdx.x]) * z * a);
            dpre[t * p.ld_dpre + p.H] = (T)(l * z);
            carry = a * l;
        }
    }
    if (p.dh0) p.dh0[(long)b * p.H + c] = carry;
}

// The gradient of an initial state that the batch shares: the rows added up in order.
__global__ __launch_bounds__(256) void scan_dh0_sum_kernel(const float* __restrict__ dh0, float* __restrict__ out, int B, int H) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= H) return;
    float s = 0.f;
    for (int b = 0; b < B; ++b) s += dh0[(long)b * H + c];
    out[c] = s;
}

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
    if (!a->B || !a->H) return STES_OK;
    STES_CHECK(a->B <= 65535, STES_ERR_UNSUPPORTED, "stes_gated_scan: more than 65535 sequences");
    STES_CHECK(a->H <= (1 << 24) && (long)a->B * ((a->H + 63) / 64) < (1L << 30), STES_ERR_UNSUPPORTED, "stes_gated_scan: too many channels");
    if (a->T) {
        STES_CHECK(a->pre && a->ld_pre >= 2L * a->H && a->bs_pre >= 0, STES_ERR_ARG, "stes_gated_scan: pre is [B][T][2H]");
        if (!bwd) STES_CHECK(a->h && apart(a->ld_h, a->T, a->bs_h, a->B, a->H), STES_ERR_ARG, "stes_gated_scan_fwd: h is [B][T][H], rows apart");
        else {
            STES_CHECK(a->states && a->dpre, STES_ERR_ARG, "stes_gated_scan_bwd: states and dpre are needed");
            STES_CHECK(apart(a->ld_dpre, a->T, a->bs_dpre, a->B, 2L * a->H), STES_ERR_ARG, "stes_gated_scan_bwd: dpre is [B][T][2H], rows apart");
            STES_CHECK(!a->dh || (a->ld_dh >= a->H && a->bs_dh >= 0), STES_ERR_ARG, "stes_gated_scan_bwd: dh is [B][T][H]");
        }
        const int64_t need = stes_gated_scan_ws_bytes(a->B, a->T, a->H);
        STES_CHECK(need == 0 || (a->ws && a->ws_bytes >= need), STES_ERR_ARG, "stes_gated_scan: workspace too small");
    }
    STES_CHECK(!a->h0 || a->bs_h0 == 0 || a->bs_h0 >= a->H, STES_ERR_ARG, "stes_gated_scan: rows of h0 overlap");
    STES_CHECK(!a->h_last || a->bs_hl >= a->H, STES_ERR_ARG, "stes_gated_scan: rows of h_last overlap");
    STES_CHECK(!(a->h_last && a->h_last == a->h0) || a->bs_h0 == a->bs_hl, STES_ERR_ARG, "stes_gated_scan: a state in place keeps its row stride");
    STES_CHECK(!a->dh0_sum || a->dh0 || !a->B, STES_ERR_ARG, "stes_gated_scan_bwd: dh0_sum needs dh0");
    return STES_OK;
}

}  // namespace

extern "C" int64_t stes_gated_scan_ws_bytes(int B, int T, int H) {
    (void)B; (void)T; (void)H;
    return 0;
}

extern "C" int stes_gated_scan_fwd(const stes_gated_scan_args* a, void* stream) {
    const int rc = scan_check(a, false);
    if (rc) return rc;
    if (!a->B || !a->H) return STES_OK;
    const dim3 grid((a->H + 63) / 64, a->B);
    if (a->f32) hipLaunchKernelGGL(scan_fwd_serial_kernel<float>, grid, dim3(64), 0, (hipStream_t)stream, *a);
    else hipLaunchKernelGGL(scan_fwd_serial_kernel<bf16>, grid, dim3(64), 0, (hipStream_t)stream, *a);
    STES_LAUNCH_CHECK();
    return STES_OK;
}

extern "C" int stes_gated_scan_bwd(const stes_gated_scan_args* a, void* stream) {
    const int rc = scan_check(a, true);
    if (rc) return rc;
    if (!a->H) return STES_OK;
    if (a->B) {
        const dim3 grid((a->H + 63) / 64, a->B);
        if (a->f32) hipLaunchKernelGGL(scan_bwd_serial_kernel<float>, grid, dim3(64), 0, (hipStream_t)stream, *a);
        else hipLaunchKernelGGL(scan_bwd_serial_kernel<bf16>, grid, dim3(64), 0, (hipStream_t)stream, *a);
        STES_LAUNCH_CHECK();
    }
    if (a->dh0_sum) {                                       // (zeros for an empty batch)
        hipLaunchKernelGGL(scan_dh0_sum_kernel, dim3((a->H + 255) / 256), dim3(256), 0, (hipStream_t)stream, a->dh0, a->dh0_sum, a->B, a->H);
        STES_LAUNCH_CHECK();
    }
    return STES_OK;
}
