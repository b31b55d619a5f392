// New tokens of packed sequences: rotary embedding of queries and keys, and keys and values into the pages of the 8-bit cache.
//
// One launch does all of it: its blocks are split between "pages" (one page, key/value head and K or V each: the scale of a page
// depends on all of its new rows, so one block sees them all; of single tokens sixteen to a block) and "queries".  A page's new rows stay in registers between the
// maximum and the rounding, so everything is read once and written once.  Bound: single tokens by latency (one launch: 128 sequences take as long
// as one); prompts by HBM with heads of 128 (eight of 4096 tokens, 807 MB: 144 to 148 us = 5.5 TB/s), and by the chain of loads before
// the first row with heads of 64, whose pages are a block's work of 8 KB (74 MB in pieces: 24.6 us = 3.0 TB/s at 56 % of the issue slots; blocks that went through
// several heads, asking for the next one's rows ahead, took 31 and 246 us: too many registers).
#include <type_traits>

#include "paged.cuh"
#include "tc_common.cuh"

namespace fmhf {
namespace {

struct AppendArgs {
    uint8_t *pages[2];       // K, V
    float *scale[2];
    long long page_stride;
    const int32_t *lengths, *table, *cu;
    long long table_stride;
    const __nv_bfloat16 *q, *x[2];       // x: K, V
    long long q_tok, q_head, x_tok[2], x_head[2];
    __nv_bfloat16 *q_out, *k_out;
    const float *cos_t, *sin_t;
    int *index;
    int B, max_pages, num_pages, n_kv, tokens, n_q, max_pos;
    unsigned page_blocks;    // blocks of the first kind
};

// PAIRS neighbouring bf16 at an address that is a multiple of 2 * PAIRS bytes (PAIRS in {4, 6, 8}), as they are and as fp32, and back.
template <int PAIRS>
__device__ __forceinline__ void load_raw(const __nv_bfloat16 *p, uint32_t (&w)[PAIRS / 2]) {
    if constexpr (PAIRS == 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (PAIRS == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < PAIRS / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
    }
}
template <int PAIRS>
__device__ __forceinline__ void to_float(const uint32_t (&w)[PAIRS / 2], float (&f)[PAIRS]) {
#pragma unroll
    for (int i = 0; i < PAIRS / 2; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <int PAIRS>
__device__ __forceinline__ void load_bf16(const __nv_bfloat16 *p, float (&f)[PAIRS]) {
    uint32_t w[PAIRS / 2];
    load_raw<PAIRS>(p, w);
    to_float<PAIRS>(w, f);
}
template <int PAIRS>
__device__ __forceinline__ void store_bf16(__nv_bfloat16 *p, const float (&f)[PAIRS]) {
    uint32_t w[PAIRS / 2];
#pragma unroll
    for (int i = 0; i < PAIRS / 2; ++i) w[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
    if constexpr (PAIRS == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (PAIRS == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    else
#pragma unroll
        for (int i = 0; i < PAIRS / 2; ++i) reinterpret_cast<uint32_t *>(p)[i] = w[i];
}
template <int PAIRS>
__device__ __forceinline__ void load_f32(const float *p, float (&f)[PAIRS]) {
#pragma unroll
    for (int i = 0; i < PAIRS / 2; ++i) {
        const float2 v = __ldg(reinterpret_cast<const float2 *>(p) + i);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
// PAIRS codes of f * inv at an address that is a multiple of PAIRS bytes (of 2 for PAIRS = 6).
template <int PAIRS, bool ALL_FINITE>
__device__ __forceinline__ void store_codes(uint8_t *p, const float (&f)[PAIRS], float inv) {
    uint32_t h[PAIRS / 2];
#pragma unroll
    for (int i = 0; i < PAIRS / 2; ++i) h[i] = to_codes2<ALL_FINITE>(f[2 * i], f[2 * i + 1], inv);
    if constexpr (PAIRS == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    else if constexpr (PAIRS == 4) *reinterpret_cast<uint32_t *>(p) = h[0] | h[1] << 16;
    else
#pragma unroll
        for (int i = 0; i < PAIRS / 2; ++i) reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)h[i];
}

// (x1, x2) turned by the angles of (c, s); products and sums are rounded one by one, as the plain expression rounds them, so that
// keys next to the border of two codes fall on the same side of it.
template <int PAIRS>
__device__ __forceinline__ void rotate(float (&x1)[PAIRS], float (&x2)[PAIRS], const float (&c)[PAIRS], const float (&s)[PAIRS]) {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const float a = x1[i], b = x2[i];
        x1[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
        x2[i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
    }
}
// The largest magnitude so far, by its bits: of every value (above kInf: there is a NaN), and of the finite ones.
constexpr uint32_t kInf = 0x7f800000u;
template <int PAIRS>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const float (&f)[PAIRS]) {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    return m;
}
template <int PAIRS>
__device__ __forceinline__ uint32_t max_finite(uint32_t m, const float (&f)[PAIRS]) {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
        m = max(m, b < kInf ? b : 0u);
    }
    return m;
}

// Rows [first, last) of the call's tokens that belong to sequence b, and what the sequence held before; both put inside the
// tensors whatever the caller's numbers say.  A negative length means that there is no sequence.
struct Piece {
    int first, last, before;
};
__device__ __forceinline__ Piece piece_of(const AppendArgs &a, int b) {
    Piece p;
    p.before = __ldg(a.lengths + b);
    p.first = a.cu ? __ldg(a.cu + b) : b;
    p.last = a.cu ? __ldg(a.cu + b + 1) : b + 1;
    if (p.first < 0 || p.last > a.tokens || p.last < p.first) {
        note_index(a.index, kPagedAppendRows);
        p.first = p.last = 0;
    }
    if (p.before < 0) p.last = p.first;
    return p;
}

// Blocks of the first kind, by their number: slot, head, K or V.  Sequence b owns the slots from cu[b] / P + 2 b on, at least as many as
// the pages that its new tokens can touch (floor((n - 1) / P) + 2 at most); which sequence a slot belongs to is a binary search.
// Eight threads a row, PASSES rows a thread, kept in registers between the maximum and the codes.  Up to 32 values are kept turned and in
// fp32; more are kept as the bf16 that were read and turned twice, at half the registers (eight prompts of 4096, heads of 128, pages of
// 128: 180 -> 162 us).  The rows are asked for before the page that they go to is known.
template <int HD, int PASSES>
__device__ void append_page(const AppendArgs &a, int log2_p, uint32_t *red) {
    constexpr int PAIRS = HD / 16;
    constexpr bool KEEP = PASSES * PAIRS <= 16;
    const int P = 1 << log2_p, kv2 = 2 * a.n_kv;
    const int slot = (int)(blockIdx.x / (unsigned)kv2), hk = (int)(blockIdx.x % (unsigned)kv2), head = hk >> 1, which = hk & 1;
    int b = 0, hi = a.B - 1;
    while (b < hi) {
        const int mid = (b + hi + 1) >> 1;
        if ((__ldg(a.cu + mid) >> log2_p) + 2 * mid <= slot) b = mid;
        else hi = mid - 1;
    }
    const int j = slot - ((__ldg(a.cu + b) >> log2_p) + 2 * b);
    const Piece pc = piece_of(a, b);
    if (pc.last <= pc.first || j < 0) return;
    // (64 bits: a length near 2^31 is the caller's mistake, not a wrap-around)
    const long long end = (long long)pc.before + (pc.last - pc.first), page_no = (long long)(pc.before >> log2_p) + j, start = page_no << log2_p;
    if (start >= end) return;
    const int had = (int)max(0ll, pc.before - start);                       // rows that are there already
    const int row_end = (int)min(min((long long)P, end - start), max(0ll, a.max_pos - start));
    const int rows_per_pass = blockDim.x >> 3, sub = threadIdx.x & 7, row0 = threadIdx.x >> 3;
    const long long tok0 = pc.first + (start - pc.before);                  // the token of the page's row 0
    const __nv_bfloat16 *x = a.x[which] + head * a.x_head[which] + sub * PAIRS;
    uint32_t w1[PASSES][PAIRS / 2], w2[PASSES][PAIRS / 2];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = row0 + i * rows_per_pass;
        if (row >= had && row < row_end) {
            const __nv_bfloat16 *src = x + (tok0 + row) * a.x_tok[which];
            load_raw<PAIRS>(src, w1[i]);
            load_raw<PAIRS>(src + HD / 2, w2[i]);
        }
    }
    const int page = page_no < a.max_pages ? __ldg(a.table + b * a.table_stride + page_no) : -1;
    if (page < 0 || page >= a.num_pages) {
        if (threadIdx.x == 0) note_index(a.index, kPagedAppendPage);
        return;
    }
    if (threadIdx.x == 0 && min((long long)P, end - start) > row_end) note_index(a.index, kPagedAppendPosition);
    float *sp = a.scale[which] + (long long)page * a.n_kv + head;
    const float old = had > 0 ? *sp : 0.f;
    float y1[KEEP ? PASSES : 1][PAIRS], y2[KEEP ? PASSES : 1][PAIRS];
    auto values = [&](int i, float (&v1)[PAIRS], float (&v2)[PAIRS]) {
        to_float<PAIRS>(w1[i], v1);
        to_float<PAIRS>(w2[i], v2);
        if (which == 0) {
            const long long pos = start + row0 + i * rows_per_pass;
            float c[PAIRS], s[PAIRS];
            load_f32<PAIRS>(a.cos_t + pos * (HD / 2) + sub * PAIRS, c);
            load_f32<PAIRS>(a.sin_t + pos * (HD / 2) + sub * PAIRS, s);
            rotate<PAIRS>(v1, v2, c, s);
        }
    };
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = row0 + i * rows_per_pass, k = KEEP ? i : 0;
        if (row >= had && row < row_end) {
            values(i, y1[k], y2[k]);
            amax = max_bits<PAIRS>(max_bits<PAIRS>(amax, y1[k]), y2[k]);
            if (which == 0 && a.k_out) {
                __nv_bfloat16 *dst = a.k_out + ((tok0 + row) * a.n_kv + head) * HD + sub * PAIRS;
                store_bf16<PAIRS>(dst, y1[k]);
                store_bf16<PAIRS>(dst + HD / 2, y2[k]);
            }
        }
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    const bool all_finite = amax < kInf;             // of this warp
    if (!all_finite) {
        amax = 0;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = row0 + i * rows_per_pass, k = KEEP ? i : 0;
            if (row >= had && row < row_end) {
                if constexpr (!KEEP) values(i, y1[k], y2[k]);
                amax = max_finite<PAIRS>(max_finite<PAIRS>(amax, y1[k]), y2[k]);
            }
        }
        amax = __reduce_max_sync(0xffffffffu, amax);
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
    __syncthreads();                                 // (every thread has read the scale, too)
    amax = __reduce_max_sync(0xffffffffu, red[threadIdx.x & (blockDim.x / 32 - 1)]);
    const float need = scale_for(amax), now = had > 0 ? fmaxf(old, need) : need;
    const float inv = inverse_scale(now);
    uint8_t *dst = a.pages[which] + page * a.page_stride + (long long)head * P * HD;
    if (threadIdx.x == 0 && row_end > had) *sp = now;
    auto store = [&](auto finite) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = row0 + i * rows_per_pass, k = KEEP ? i : 0;
            if (row >= had && row < row_end) {
                if constexpr (!KEEP) values(i, y1[k], y2[k]);
                store_codes<PAIRS, decltype(finite)::value>(dst + row * HD + sub * PAIRS, y1[k], inv);
                store_codes<PAIRS, decltype(finite)::value>(dst + row * HD + HD / 2 + sub * PAIRS, y2[k], inv);
            }
        }
    };
    if (all_finite) store(std::true_type{});
    else store(std::false_type{});
    if (had > 0 && now != old) {
        const float ratio = old * inv;
        for (int i = threadIdx.x; i < had * (HD / 16); i += blockDim.x) {
            uint4 *c = reinterpret_cast<uint4 *>(dst) + i;
            const uint4 v = *c;
            *c = make_uint4(rescale4(v.x, ratio), rescale4(v.y, ratio), rescale4(v.z, ratio), rescale4(v.w, ratio));
        }
    }
}

// One token a sequence: eight threads a (sequence, head, K or V).  The page's other rows are touched only where its scale grows.
template <int HD>
__device__ void append_token(const AppendArgs &a, int log2_p) {
    constexpr int PAIRS = HD / 16;
    const long long it = (long long)blockIdx.x * (blockDim.x >> 3) + (threadIdx.x >> 3);
    const int sub = threadIdx.x & 7, which = (int)(it & 1), head = (int)((it >> 1) % a.n_kv);
    const unsigned group = 0xffu << (threadIdx.x & 24);
    const long long b = (it >> 1) / a.n_kv;
    if (b >= a.B) return;
    // (the row is asked for before its place is known)
    float y1[PAIRS], y2[PAIRS];
    const __nv_bfloat16 *src = a.x[which] + b * a.x_tok[which] + head * a.x_head[which] + sub * PAIRS;
    load_bf16<PAIRS>(src, y1);
    load_bf16<PAIRS>(src + HD / 2, y2);
    const int pos = __ldg(a.lengths + b);
    if (pos < 0) return;
    const int P = 1 << log2_p, page_no = pos >> log2_p, row = pos & (P - 1);
    const int page = page_no < a.max_pages ? __ldg(a.table + b * a.table_stride + page_no) : -1;
    if (page < 0 || page >= a.num_pages || pos >= a.max_pos) {
        note_index(a.index, page < 0 || page >= a.num_pages ? kPagedAppendPage : kPagedAppendPosition);
        return;
    }
    float *sp = a.scale[which] + (long long)page * a.n_kv + head;
    const float old = *sp;
    if (which == 0) {
        float c[PAIRS], s[PAIRS];
        load_f32<PAIRS>(a.cos_t + (long long)pos * (HD / 2) + sub * PAIRS, c);
        load_f32<PAIRS>(a.sin_t + (long long)pos * (HD / 2) + sub * PAIRS, s);
        rotate<PAIRS>(y1, y2, c, s);
        if (a.k_out) {
            __nv_bfloat16 *dst = a.k_out + (b * a.n_kv + head) * HD + sub * PAIRS;
            store_bf16<PAIRS>(dst, y1);
            store_bf16<PAIRS>(dst + HD / 2, y2);
        }
    }
    uint32_t amax = max_finite<PAIRS>(max_finite<PAIRS>(0, y1), y2);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(group, amax, o));
    const float need = scale_for(amax), now = row > 0 ? fmaxf(old, need) : need, inv = inverse_scale(now);
    uint8_t *dst = a.pages[which] + page * a.page_stride + (long long)head * P * HD;
    __syncwarp(group);                           // all eight have read the scale
    if (sub == 0 && now != old) *sp = now;
    store_codes<PAIRS, false>(dst + row * HD + sub * PAIRS, y1, inv);
    store_codes<PAIRS, false>(dst + row * HD + HD / 2 + sub * PAIRS, y2, inv);
    if (row > 0 && now != old) {
        const float ratio = old * inv;
#pragma unroll 4
        for (int i = sub; i < row * (HD / 16); i += 8) {
            uint4 *c = reinterpret_cast<uint4 *>(dst) + i;
            const uint4 v = *c;
            *c = make_uint4(rescale4(v.x, ratio), rescale4(v.y, ratio), rescale4(v.z, ratio), rescale4(v.w, ratio));
        }
    }
}

// Which sequence a token belongs to (the last b with cu[b] <= t), and its position; -1 where it has none.
__device__ __forceinline__ long long position_of(const AppendArgs &a, int t) {
    int b = t;
    if (a.cu) {
        int lo = 0, hi = a.B - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (__ldg(a.cu + mid) <= t) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
    }
    const Piece pc = piece_of(a, b);
    return t >= pc.first && t < pc.last ? (long long)pc.before + (t - pc.first) : -1;
}

// Blocks of the second kind: eight threads hold the sines and cosines of a token and turn up to eight of its heads with them.
constexpr int kHeadsPerThread = 8;
template <int HD>
__device__ void append_queries(const AppendArgs &a) {
    constexpr int PAIRS = HD / 16;
    const int groups = (a.n_q + kHeadsPerThread - 1) / kHeadsPerThread;
    const long long it = (long long)(blockIdx.x - a.page_blocks) * (blockDim.x >> 3) + (threadIdx.x >> 3);
    const int sub = threadIdx.x & 7, h0 = (int)(it % groups) * kHeadsPerThread;
    const long long t = it / groups;
    if (t >= a.tokens) return;
    const long long pos = position_of(a, (int)t);
    if (pos < 0) return;
    if (pos >= a.max_pos) {
        note_index(a.index, kPagedAppendPosition);
        return;
    }
    float c[PAIRS], s[PAIRS];
    load_f32<PAIRS>(a.cos_t + pos * (HD / 2) + sub * PAIRS, c);
    load_f32<PAIRS>(a.sin_t + pos * (HD / 2) + sub * PAIRS, s);
#pragma unroll 4
    for (int h = h0; h < min(h0 + kHeadsPerThread, a.n_q); ++h) {
        const __nv_bfloat16 *src = a.q + t * a.q_tok + h * a.q_head + sub * PAIRS;
        float x1[PAIRS], x2[PAIRS];
        load_bf16<PAIRS>(src, x1);
        load_bf16<PAIRS>(src + HD / 2, x2);
        rotate<PAIRS>(x1, x2, c, s);
        __nv_bfloat16 *dst = a.q_out + (t * a.n_q + h) * HD + sub * PAIRS;
        store_bf16<PAIRS>(dst, x1);
        store_bf16<PAIRS>(dst + HD / 2, x2);
    }
}

// PASSES: rows of a page that a thread takes; 0: one token a sequence.  Blocks that an SM is to hold, against the compiler's choice: eight prompts
// of 4096 tokens, heads of 128 in pages of 128 (three blocks, not two) 153 -> 144 us, of 64 (four, not three) 145 -> 139.
template <int HD, int PASSES>
constexpr int kMinBlocks = HD == 64 ? 5 : HD == 128 && PASSES == 4 ? 3 : 4;
template <int HD, int PASSES>
__global__ void __launch_bounds__(256, kMinBlocks<HD, PASSES>) paged_append_kernel(const AppendArgs a, int log2_p) {
    __shared__ uint32_t red[8];
    if (blockIdx.x >= a.page_blocks) append_queries<HD>(a);
    else if constexpr (PASSES > 0) append_page<HD, PASSES>(a, log2_p, red);
    else append_token<HD>(a, log2_p);
}

}  // namespace

int paged_append(const flashmhf_paged_append_params &p, const DeviceCtl &ctl, cudaStream_t st, int *n_launch) {
    AppendArgs a{};
    const flashmhf_kv_pages &g = p.pages;
    a.pages[0] = static_cast<uint8_t *>(g.k); a.pages[1] = static_cast<uint8_t *>(g.v);
    a.scale[0] = g.k_scale; a.scale[1] = g.v_scale;
    a.page_stride = g.page_stride;
    a.lengths = p.seq.lengths; a.table = p.seq.table; a.cu = p.cu_seqlens;
    a.table_stride = p.seq.table_stride;
    a.q = static_cast<const __nv_bfloat16 *>(p.q);
    a.x[0] = static_cast<const __nv_bfloat16 *>(p.k); a.x[1] = static_cast<const __nv_bfloat16 *>(p.v);
    a.q_tok = p.q_stride[0]; a.q_head = p.q_stride[1];
    a.x_tok[0] = p.k_stride[0]; a.x_head[0] = p.k_stride[1];
    a.x_tok[1] = p.v_stride[0]; a.x_head[1] = p.v_stride[1];
    a.q_out = static_cast<__nv_bfloat16 *>(p.q_out);
    a.k_out = static_cast<__nv_bfloat16 *>(p.k_out);
    a.cos_t = p.cos_t; a.sin_t = p.sin_t;
    a.index = ctl.index;
    a.B = p.seq.B; a.max_pages = p.seq.max_pages; a.num_pages = g.num_pages; a.n_kv = g.n_kv;
    a.tokens = p.tokens; a.n_q = p.q ? p.n_q : 0; a.max_pos = p.max_positions;
    const int P = g.page_size, threads = a.cu ? (P * 8 < 256 ? P * 8 : 256) : 128;
    const long long page_blocks = a.cu ? ((long long)p.tokens / P + 2ll * a.B) * 2 * a.n_kv : ((long long)a.B * 2 * a.n_kv + 15) / 16;
    const long long groups = a.n_q ? (a.n_q + kHeadsPerThread - 1) / kHeadsPerThread : 0, per_block = threads / 8;
    const long long blocks = page_blocks + ((long long)p.tokens * groups + per_block - 1) / per_block;
    if (blocks > 0x7fffffffll) return FLASHMHF_ERR_BAD_SHAPE;
    a.page_blocks = (unsigned)page_blocks;
    auto choose = [&](auto k0, auto k1, auto k2, auto k4) { return !a.cu ? k0 : P == 128 ? k4 : P == 64 ? k2 : k1; };
    auto kernel = g.head_dim == 64   ? choose(paged_append_kernel<64, 0>, paged_append_kernel<64, 1>, paged_append_kernel<64, 2>, paged_append_kernel<64, 4>)
                  : g.head_dim == 96 ? choose(paged_append_kernel<96, 0>, paged_append_kernel<96, 1>, paged_append_kernel<96, 2>, paged_append_kernel<96, 4>)
                                     : choose(paged_append_kernel<128, 0>, paged_append_kernel<128, 1>, paged_append_kernel<128, 2>, paged_append_kernel<128, 4>);
    const cudaError_t e = launch_kernel(false, kernel, dim3((unsigned)blocks), dim3(threads), 0, st, a, __builtin_ctz((unsigned)P));
    if (e != cudaSuccess) {
        set_cuda_error(e, "paged append launch");
        return FLASHMHF_ERR_CUDA;
    }
    ++*n_launch;
    return FLASHMHF_OK;
}

}  // namespace fmhf
