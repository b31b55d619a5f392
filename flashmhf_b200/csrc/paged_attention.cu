// Attention of the newest tokens of each sequence over its pages of the 8-bit cache.
#include "paged.cuh"

namespace fmhf {
namespace {

struct PagedArgs {
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    long long page_stride;
    const int32_t *lengths, *table;
    long long table_stride;
    const __nv_bfloat16 *q;
    __nv_bfloat16 *o;
    long long q_stride[3], o_stride[3];
    float *lse;
    int *status;
    int B, max_pages, num_pages, n_kv, n_q, n_new, P;
    float scale;
};

__device__ __forceinline__ float code_value(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

// One warp a row (sequence, new token, query head); lane l holds the output's elements l, l + 32, ...
template <int HD>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedArgs a) {
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (long long)a.B * a.n_new * a.n_q) return;
    const int h = (int)(row % a.n_q), i = (int)(row / a.n_q % a.n_new), b = (int)(row / a.n_q / a.n_new), kh = h / (a.n_q / a.n_kv);
    float q[N], o[N] = {};
#pragma unroll
    for (int n = 0; n < N; ++n)
        q[n] = __bfloat162float(a.q[b * a.q_stride[0] + i * a.q_stride[1] + h * a.q_stride[2] + n * 32 + lane]);
    long long len = a.lengths[b];
    if (len > (long long)a.max_pages * a.P) {
        note_index(a.status, kPagedAttnLength);
        len = (long long)a.max_pages * a.P;
    }
    len -= a.n_new - 1 - i;
    float m = -INFINITY, l = 0.f;
    for (long long p = 0; p < len; ++p) {
        const int page = a.table[b * a.table_stride + p / a.P];
        if (page < 0 || page >= a.num_pages) {
            note_index(a.status, kPagedAttnPage);
            continue;
        }
        const long long at = page * a.page_stride + ((long long)kh * a.P + p % a.P) * HD + lane;
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) s += q[n] * code_value(a.k[at + n * 32]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= a.k_scale[(long long)page * a.n_kv + kh] * a.scale;
        const float now = fmaxf(m, s), keep = expf(m - now), w = expf(s - now), wv = w * a.v_scale[(long long)page * a.n_kv + kh];
        m = now;
        l = l * keep + w;
#pragma unroll
        for (int n = 0; n < N; ++n) o[n] = o[n] * keep + wv * code_value(a.v[at + n * 32]);
    }
    const float r = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
        a.o[b * a.o_stride[0] + i * a.o_stride[1] + h * a.o_stride[2] + n * 32 + lane] = __float2bfloat16(o[n] * r);
    if (a.lse && lane == 0) a.lse[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace

size_t paged_attention_workspace_bytes(const flashmhf_paged_attention_params &) { return 0; }

int paged_attention(const flashmhf_paged_attention_params &p, const DeviceCtl &ctl, cudaStream_t st, int *n_launch) {
    PagedArgs a{};
    const flashmhf_kv_pages &g = p.pages;
    a.k = static_cast<const uint8_t *>(g.k); a.v = static_cast<const uint8_t *>(g.v);
    a.k_scale = g.k_scale; a.v_scale = g.v_scale; a.page_stride = g.page_stride;
    a.lengths = p.seq.lengths; a.table = p.seq.table; a.table_stride = p.seq.table_stride;
    a.q = static_cast<const __nv_bfloat16 *>(p.q); a.o = static_cast<__nv_bfloat16 *>(p.o);
    for (int i = 0; i < 3; ++i) { a.q_stride[i] = p.q_stride[i]; a.o_stride[i] = p.o_stride[i]; }
    a.lse = p.lse; a.status = ctl.status;
    a.B = p.seq.B; a.max_pages = p.seq.max_pages; a.num_pages = g.num_pages; a.n_kv = g.n_kv; a.n_q = p.n_q; a.n_new = p.n_new; a.P = g.page_size;
    a.scale = p.scale;
    const long long rows = (long long)a.B * a.n_new * a.n_q;
    if ((rows + 3) / 4 > 0x7fffffffll) return FLASHMHF_ERR_BAD_SHAPE;
    auto kernel = g.head_dim == 64 ? paged_attention_kernel<64> : g.head_dim == 96 ? paged_attention_kernel<96> : paged_attention_kernel<128>;
    const cudaError_t e = launch_kernel(false, kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a);
    if (e != cudaSuccess) {
        set_cuda_error(e, "paged attention launch");
        return FLASHMHF_ERR_CUDA;
    }
    ++*n_launch;
    return FLASHMHF_OK;
}

}  // namespace fmhf
