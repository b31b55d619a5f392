// Attention over packed prompts.
#include "paged.cuh"

namespace fmhf {
namespace {

struct PromptArgs {
    const __nv_bfloat16 *q, *k, *v;
    __nv_bfloat16 *o;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
    float *lse;
    const int32_t *cu_q, *cu_k;
    int *status;
    int B, tokens_q, tokens_k, n_q, n_kv, causal;
    float scale;
};

// One warp a row (token, query head); lane l holds the output's elements l, l + 32, ...
template <int HD>
__global__ void __launch_bounds__(128) prompt_attention_kernel(const PromptArgs a) {
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (long long)a.tokens_q * a.n_q) return;
    const int h = (int)(row % a.n_q), t = (int)(row / a.n_q), kh = h / (a.n_q / a.n_kv);
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu_q[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    const int q0 = a.cu_q[lo], q1 = a.cu_q[lo + 1], k0 = a.cu_k[lo], k1 = a.cu_k[lo + 1];
    if (t < q0 || t >= q1) return;
    if (q0 < 0 || q1 > a.tokens_q || k0 < 0 || k1 > a.tokens_k || k1 < k0) {
        note_index(a.status, kPromptRows);
        return;
    }
    const int lk = k1 - k0, see = a.causal ? min(lk, t - q0 + 1 + lk - (q1 - q0)) : lk;
    float q[N], o[N] = {};
#pragma unroll
    for (int n = 0; n < N; ++n) q[n] = __bfloat162float(a.q[t * a.q_tok + h * a.q_head + n * 32 + lane]);
    float m = -INFINITY, l = 0.f;
    for (int c = 0; c < see; ++c) {
        const __nv_bfloat16 *k = a.k + (long long)(k0 + c) * a.k_tok + kh * a.k_head + lane, *v = a.v + (long long)(k0 + c) * a.v_tok + kh * a.v_head + lane;
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) s += q[n] * __bfloat162float(k[n * 32]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= a.scale;
        const float now = fmaxf(m, s), keep = expf(m - now), w = expf(s - now);
        m = now;
        l = l * keep + w;
#pragma unroll
        for (int n = 0; n < N; ++n) o[n] = o[n] * keep + w * __bfloat162float(v[n * 32]);
    }
    const float r = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) a.o[(long long)t * a.o_tok + h * a.o_head + n * 32 + lane] = __float2bfloat16(o[n] * r);
    if (a.lse && lane == 0) a.lse[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace

int prompt_attention(const flashmhf_prompt_attention_params &p, const DeviceCtl &ctl, cudaStream_t st, int *n_launch) {
    PromptArgs a{};
    a.q = static_cast<const __nv_bfloat16 *>(p.q); a.k = static_cast<const __nv_bfloat16 *>(p.k); a.v = static_cast<const __nv_bfloat16 *>(p.v);
    a.o = static_cast<__nv_bfloat16 *>(p.o);
    a.q_tok = p.q_stride[0]; a.q_head = p.q_stride[1]; a.k_tok = p.k_stride[0]; a.k_head = p.k_stride[1];
    a.v_tok = p.v_stride[0]; a.v_head = p.v_stride[1]; a.o_tok = p.o_stride[0]; a.o_head = p.o_stride[1];
    a.lse = p.lse; a.cu_q = p.cu_q; a.cu_k = p.cu_k; a.status = ctl.status;
    a.B = p.B; a.tokens_q = p.tokens_q; a.tokens_k = p.tokens_k; a.n_q = p.n_q; a.n_kv = p.n_kv; a.causal = p.causal; a.scale = p.scale;
    const long long rows = (long long)a.tokens_q * a.n_q;
    if ((rows + 3) / 4 > 0x7fffffffll) return FLASHMHF_ERR_BAD_SHAPE;
    auto kernel = p.head_dim == 64 ? prompt_attention_kernel<64> : p.head_dim == 96 ? prompt_attention_kernel<96> : prompt_attention_kernel<128>;
    const cudaError_t e = launch_kernel(false, kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a);
    if (e != cudaSuccess) {
        set_cuda_error(e, "prompt attention launch");
        return FLASHMHF_ERR_CUDA;
    }
    ++*n_launch;
    return FLASHMHF_OK;
}

}  // namespace fmhf
