// Attention of the newest tokens of each sequence over its pages of the 8-bit cache.
//
// A code that is read is used by up to eight query rows (the query heads of a key/value head, times the new tokens), so the call
// is bound by HBM as soon as the cache is larger than a few MB; below that by the chain of dependent loads (lengths, page numbers,
// scales, codes) and its two launches.  More than eight rows a key/value head read the cache once for each eight of them: 64 sequences of 8192, 32 / 8 heads
// of 128, take 176 us with one new token, 187 with two, 345 with four and 655 with eight.
//
// Splitting.  The tokens of all (sequence, key/value head, eight query rows) are laid end to end in units of 64 and dealt out to all warps of the
// GPU in equal contiguous runs, by lengths that only the device knows: one long sequence and a hundred short ones load the machine alike.
// A warp works alone: its codes come by bulk copies into a ring of its own in shared memory (16 KB a warp, 192 KB on an SM, or 18 and 216
// with heads of 96: what 6.5 TB/s at over a microsecond's latency take), and go from there into fragments, 32 tokens at a time: two chains of products, one look at the
// maximum.  64 sequences of 8192 tokens, 8 heads of 128 (1.07 GB): 176 to 187 us from GPU to GPU = 5.7 to 6.1 TB/s; 64 of 4096, 32 heads of 64: 176 us; two of 65537, 4 heads of
// 128: 39 us.  In registers, 16 tokens ahead: 224, -, 61.  Sixteen warps with 12 KB and 16 tokens at a time: 179, 203, 43; eight with 24 KB: 188,
// 204, 38, and 25 instead of 21 us for 32 ragged sequences.  Copies that run on into the next segment of a run: 187, 213, 45 (more instructions a stage
// than the waits that they save).
// A run that covers all of an item writes its rows; else the warp writes its part (at most two a warp: the ends of its run) with its maximum
// and sum, and a second kernel adds the parts in the order of the tokens.
//
// Products.  16 tokens at a time, on mma.m16n8k16 in fp16 with fp32 accumulators: S^T = K Q^T (tokens x rows), O^T += V^T P^T
// (dims x rows): tokens and dims fill the 16 of a tile, and the few query rows its 8 columns (tcgen05 tiles have at least 64 or 128 of
// them, and one operand of each product would have to be converted into shared memory).  e4m3 is exact in fp16; queries are scaled by a power of two so that their
// largest is between 2^14 and 2^15: exact down to 2^-28 of it.  P is rounded to 11 bits; maxima, sums and O are fp32.
// Which dims a lane's share of a fragment stands for is free as long as both operands agree, so a lane loads HD / 4 neighbouring codes of a
// key and HD / 8 of a value, straight into fragments; pairs of tokens that V needs side by side are made by byte permutation.
#include <atomic>

#include "paged.cuh"
#include "tc_common.cuh"

namespace fmhf {
namespace {

constexpr int kUnit = 64;            // tokens
constexpr int kCols = 8;             // query rows of an item
constexpr int kWarps = 4;            // of a block; they have nothing to do with one another
constexpr int kKernelPaged = 7;      // status codes 701..
template <int HD>
struct Ring {
    static constexpr int kTokens = HD == 64 ? 64 : 32, kStages = HD == 96 ? 3 : 2, kBlocks = 3;       // tokens of a stage, stages, blocks on an SM
    static constexpr uint32_t kHalf = kTokens * HD, kStage = 2 * kHalf;                 // keys, then values
    static constexpr uint32_t kBytes = kStages * kStage;
};
// Weights are kept as P = 2^(s + e - m), 2^e the scale of the values' page: P V is then a product of P and bare codes.  m is set so that the
// largest P is 2^7, and set again when one exceeds 2^15: fp16 holds P to 11 bits down to 2^-21 of the largest product of weight and
// scale, and in steps of 2^-31 of it below.  e is kept within +-45 (what a scale is beyond that multiplies the product instead), so that
// the sum of the weights themselves, P 2^-e, loses nothing in fp32 to pages whose values are larger.
// Where the scales of the pages that a run knows (32 to 64 ahead) are more than 2^8 apart, P of the smaller ones would lose its bits to the larger ones'
// m, though other dimensions may hold nothing but theirs.  There the weights of 16 tokens have an m of their own, which puts their largest between 2^6 and
// 2^7; what it differs from the run's multiplies their product in fp32, as the rest of a scale does that is not a power of two or beyond
// 2^+-45: 64 sequences of 8192 tokens, every other page 2^16 larger, 242 us instead of 176.  Either way a weight is off by 2^-11 of itself, or by 2^-24 of the row's largest.
constexpr float kTop = 7.f, kLazyMax = 15.f;
constexpr int kMaxExp = 45, kFar = 8;

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
    float *part;                     // [worker][2][kCols][HD] sums of a warp's parts
    float2 *ml;                      // [worker][2][kCols] their maxima and sums of weights
    int4 *shared_by;                 // [item]: first and last worker of it, and which part of the first one's
    int *index;
    int B, max_pages, num_pages, n_kv, n_q, n_new, log_page, group, col_tiles, workers;
    float c;                         // scale * log2(e)
    WaitArgs wait;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half_pair(uint32_t two_codes) {      // the codes in the lower 16 bits
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two_codes));
    return r;
}
__device__ __forceinline__ uint32_t half_pair_hi(uint32_t codes) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(codes));
    return r;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t r) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(r));
    return d;
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// W words from an address that is a multiple of 4 W bytes where W is a power of two, of 8 for W = 6, of 4 for W = 3.
template <int W>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[W]) {
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const uint4 v = *(reinterpret_cast<const uint4 *>(p) + i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (W % 2 == 0) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            const uint2 v = *(reinterpret_cast<const uint2 *>(p) + i);
            w[2 * i] = v.x; w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = *(reinterpret_cast<const uint32_t *>(p) + i);
    }
}

// Tokens in the cache of sequence b, as far as its row of the table goes.
__device__ __forceinline__ int length_of(const PagedArgs &a, int b) {
    const int n = __ldg(a.lengths + b);
    const long long most = (long long)a.max_pages << a.log_page;
    if (n > most) note_index(a.index, kPagedAttnLength);
    return max(0, (int)min((long long)n, most));
}
__device__ __forceinline__ long long units_of(int len) { return (len + kUnit - 1) / kUnit; }
__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Units of an item of each sequence, summed over sequences first .. last - 1 (a whole warp asks).
__device__ long long units_between(const PagedArgs &a, int first, int last) {
    long long n = 0;
    for (int b = first + (threadIdx.x & 31); b < last; b += 32) n += units_of(length_of(a, b));
    return warp_sum(n);
}

// Units dealt out: worker w has first(w) .. first(w + 1) - 1; the first `extra` workers have one more than the others, and every worker has one.
struct Deal {
    int workers, extra;
    long long each;
    __device__ Deal(long long total, int most) {
        workers = (int)min((long long)most, total);
        const long long w = max(workers, 1);
        each = divide(total, w);
        extra = (int)(total - each * w);
    }
    // 32-bit division where it fits: the 64-bit one is a hundred instructions
    static __device__ __forceinline__ long long divide(long long a, long long b) {
        return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
    }
    __device__ __forceinline__ long long first(int w) const { return w * each + min(w, extra); }
    __device__ __forceinline__ int owner(long long unit) const {
        const long long cut = extra * (each + 1);
        return (int)(unit < cut ? divide(unit, each + 1) : extra + divide(unit - cut, each));
    }
};

// What a stage's pages stand for, by its 16 tokens: key scale (NaN: no page), exponent of the value scale (clamped), the rest of that scale;
// `plain`: that is 1, and the run's scales are not far apart.
struct Granule {
    float ks, ve, vr;
    int plain;
};

template <int HD>
__global__ void __launch_bounds__(kWarps * 32, Ring<HD>::kBlocks) paged_attention_kernel(const PagedArgs a) {
    using R = Ring<HD>;
    constexpr int KK = HD / 16, MT = HD / 16, NS = R::kStages, NG = R::kTokens / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) unsigned long long bars[kWarps][NS];
    __shared__ Granule granules[kWarps][NS][NG];
    __shared__ int2 spans[kWarps];      // least and largest exponent of the values' scales, of the pages that a warp's run knows so far
    __shared__ int abort_flag;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int worker = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int warp = threadIdx.x >> 5;
    const uint8_t *ring = smem + warp * R::kBytes;
    const uint32_t ring_at = smem_u32(ring), bar_at = smem_u32(&bars[warp][0]);
    const WaitCtl ctl{&abort_flag, a.wait};
    // (asked for before anything that waits: the first of a chain of loads)
    const int first_len = lane < a.B ? length_of(a, lane) : 0;
    if (threadIdx.x == 0) abort_flag = launch_aborted(a.wait);
    if (lane < NS) mbar_init(bar_at + 8 * lane, 1);
    fence_mbar_init();
    __syncthreads();
    griddep_launch_dependents();
    if (abort_flag) return;
    uint32_t issued = 0, used = 0;      // stages, counted through all of the run
    const int per_seq = a.n_kv * a.col_tiles, P = 1 << a.log_page, rows = a.group * a.n_new;
    const Deal deal((warp_sum(units_of(first_len)) + (a.B > 32 ? units_between(a, 32, a.B) : 0)) * per_seq, a.workers);
    if (worker >= deal.workers) return;
    long long u = deal.first(worker);
    const long long u_end = deal.first(worker + 1), u_first = u;

    // the sequence that unit u belongs to, and where its units begin
    int b = 0;
    long long base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        const long long n = units_of(b0 == 0 ? first_len : b0 + lane < a.B ? length_of(a, b0 + lane) : 0) * per_seq;
        long long sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + sum > u);
        if (past) {
            const int at = __ffs(past) - 1;
            b = b0 + at;
            base += __shfl_sync(0xffffffffu, sum - n, at);
            break;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }

    while (u < u_end) {
        int len = length_of(a, b);
        long long n_units = units_of(len);
        while (u >= base + n_units * per_seq) {         // (sequences without tokens are passed over)
            base += n_units * per_seq;
            len = length_of(a, ++b);
            n_units = units_of(len);
        }
        const int item = (int)Deal::divide(u - base, n_units), head = item / a.col_tiles, col0 = (item % a.col_tiles) * kCols;
        const long long begin = base + item * n_units, end = begin + n_units, stop = min(end, u_end);
        const int tok0 = (int)(u - begin) * kUnit, tok1 = (int)min((long long)len, (stop - begin) * kUnit);

        // tokens that the lane's columns see
        int see[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) see[i] = len - (a.n_new - 1 - min(rows - 1, col0 + 2 * t + i) / a.group);
        const int all = len - (a.n_new - 1);

        // queries: column g of the tile, dims HD / 4 * t on (asked for here, put into fragments when the codes are on their way)
        uint32_t raw_q[HD / 8] = {};
        if (col0 + g < rows) {
            const int r = col0 + g;
            load_words<HD / 8>(reinterpret_cast<const uint8_t *>(a.q + b * a.q_stride[0] + (r / a.group) * a.q_stride[1] +
                                                                 (head * a.group + r % a.group) * a.q_stride[2] + t * (HD / 4)), raw_q);
        }

        // pages: lane i knows page first_page + i and its scales, and those of the 32 after
        const int32_t *table = a.table + b * a.table_stride;
        const int last_page = (tok1 - 1) >> a.log_page;
        int page_base = tok0 >> a.log_page;
        int id, id2;
        float ks, vs, ks2, vs2;
        auto pages = [&](int first, int &pid, float &k, float &v) {
            pid = first + lane <= last_page ? __ldg(table + first + lane) : -1;
            if (first + lane <= last_page && (pid < 0 || pid >= a.num_pages)) {
                note_index(a.index, kPagedAttnPage);
                pid = -1;
            }
            const long long at = (long long)max(pid, 0) * a.n_kv + head;      // (of no page: any scale)
            k = __ldg(a.k_scale + at);
            v = __ldg(a.v_scale + at);
        };
        pages(page_base, id, ks, vs);
        float o[MT][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        // Copies of the stage of tokens from `tok` on.  The warp has read what was there (it meets before each call).  Lane 2 i copies the keys and
        // lane 2 i + 1 the values of the stage's i-th page (or of the stage, where a page holds more); lane i writes down the scales of its i-th 16.
        auto load = [&](int tok) {
            const uint32_t st = issued++ % NS, dst = ring_at + st * R::kStage, bar = bar_at + 8 * st;
            const int n = min(R::kTokens, (tok1 - tok + 15) & ~15), step = min(P, R::kTokens), page = tok >> a.log_page;      // (rows of a page exist, used or not)
            const bool more = page - page_base >= 32;
            if (more) {        // (pages come in whole stages)
                id = id2; ks = ks2; vs = vs2;
                page_base += 32;
                pages(page_base + 32, id2, ks2, vs2);
            }
            const int from = (lane >> 1) * step, at_copy = (from >> a.log_page) + page - page_base, at_scale = ((tok + lane * 16) >> a.log_page) - page_base;
            const int pid = __shfl_sync(0xffffffffu, id, at_copy & 31), gid = __shfl_sync(0xffffffffu, id, at_scale & 31);
            const float k = __shfl_sync(0xffffffffu, ks, at_scale & 31), v = __shfl_sync(0xffffffffu, vs, at_scale & 31);
            const bool copies = from < n && pid >= 0;
            const uint32_t size = copies ? (uint32_t)min(step, n - from) * HD : 0;
            const uint32_t bytes = __reduce_add_sync(0xffffffffu, size);
            if (lane == 0) {
                if (bytes) mbar_arrive_expect_tx(bar, bytes);
                else mbar_arrive(bar);
            }
            __syncwarp();
            if (copies) {
                const long long at = (long long)pid * a.page_stride + ((long long)head * P + ((tok + from) & (P - 1))) * HD;
                bulk_load(dst + (lane & 1) * R::kHalf + from * HD, (lane & 1 ? a.v : a.k) + at, size, bar);
            }
            // (after the copies: they do not wait for the scales)
            auto exponent = [](float scale) { return min(max((int)(__float_as_uint(scale) >> 23 & 255) - 127, -kMaxExp), kMaxExp); };
            if (more || tok == tok0) {
                const int ev = exponent(vs), least = __reduce_min_sync(0xffffffffu, id >= 0 ? ev : kMaxExp), most = __reduce_max_sync(0xffffffffu, id >= 0 ? ev : -kMaxExp);
                if (lane == 0) spans[warp] = more ? make_int2(min(spans[warp].x, least), max(spans[warp].y, most)) : make_int2(least, most);
                __syncwarp();
            }
            if (lane < NG) {
                const int e = exponent(v);
                const float vr = v * __uint_as_float((uint32_t)(127 - e) << 23);
                granules[warp][st][lane] = lane * 16 < n && gid >= 0 ? Granule{k, (float)e, vr, vr == 1.f && spans[warp].y - spans[warp].x <= kFar}
                                                                     : Granule{NAN, 0.f, 1.f, 1};
            }
        };
        for (int i = 0; i < NS; ++i)
            if (tok0 + i * R::kTokens < tok1) load(tok0 + i * R::kTokens);
        __syncwarp();
        pages(page_base + 32, id2, ks2, vs2);      // (a few stages do not reach them)
        uint32_t qf[KK][2];
        float fac[2];                                    // what scores of columns 2t, 2t + 1 are multiplied by
        {
            float x[HD / 4], top = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                x[2 * i] = __uint_as_float(raw_q[i] << 16);
                x[2 * i + 1] = __uint_as_float(raw_q[i] & 0xffff0000u);
            }
#pragma unroll
            for (int i = 0; i < HD / 4; ++i) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^14 over the power of two in `top`, and its inverse; both normal numbers (top below 2^-112 loses bits that no score shows)
            const int e = min(max((int)(__float_as_uint(top) >> 23), 15), 254);
            const float up = __uint_as_float((uint32_t)(254 + 14 - e) << 23), down = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
            for (int i = 0; i < KK; ++i) {
                qf[i][0] = pack_half(x[4 * i] * up, x[4 * i + 1] * up);
                qf[i][1] = pack_half(x[4 * i + 2] * up, x[4 * i + 3] * up);
            }
            fac[0] = a.c * __shfl_sync(0xffffffffu, down, 8 * t);
            fac[1] = a.c * __shfl_sync(0xffffffffu, down, 8 * t + 4);
        }
        // 32 tokens: two chains of products, one look at the maximum.
        auto compute = [&](int tok, const uint8_t *keys, const Granule *gr) {
            const Granule st[2] = {gr[0], gr[1]};
            float s[2][4] = {};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t k0[HD / 16], k1[HD / 16];
                load_words<HD / 16>(keys + (16 * x + g) * HD + t * (HD / 4), k0);
                load_words<HD / 16>(keys + (16 * x + g + 8) * HD + t * (HD / 4), k1);
#pragma unroll
                for (int i = 0; i < KK; ++i) mma16(s[x], half_pair(k0[i]), half_pair(k1[i]), half_pair_hi(k0[i]), half_pair_hi(k1[i]), qf[i][0], qf[i][1]);
            }
            uint32_t v[2][4][HD / 32];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) load_words<HD / 32>(keys + R::kHalf + (16 * x + 2 * t + (i & 1) + 8 * (i >> 1)) * HD + g * (HD / 8), v[x][i]);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float f0 = fac[0] * st[x].ks, f1 = fac[1] * st[x].ks;
                s[x][0] = fmaf(s[x][0], f0, st[x].ve); s[x][1] = fmaf(s[x][1], f1, st[x].ve);
                s[x][2] = fmaf(s[x][2], f0, st[x].ve); s[x][3] = fmaf(s[x][3], f1, st[x].ve);
            }
            if (tok + 32 > min(all, tok1) || st[0].ks != st[0].ks || st[1].ks != st[1].ks) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    // tokens of the 16 that are there (of no page: none); what lies behind them may be anything
                    const bool none = st[x].ks != st[x].ks;
                    const int from = tok + 16 * x, left = none ? 0 : tok1 - from;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (none || from + g + 8 * (i >> 1) >= min(see[i & 1], tok1)) s[x][i] = -INFINITY;
                        if (2 * t + (i & 1) + 8 * (i >> 1) >= left)
#pragma unroll
                            for (int w = 0; w < HD / 32; ++w) v[x][i][w] = 0;
                    }
                }
            }
            const float x0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])), x1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
            if (__any_sync(0xffffffffu, x0 - m[0] > kLazyMax || x1 - m[1] > kLazyMax)) {
                float n0 = x0, n1 = x1;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, d));
                    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, d));
                }
                // (a column whose maximum has not grown, or that has seen nothing, keeps what it has)
                n0 = n0 - kTop > m[0] ? n0 - kTop : m[0];
                n1 = n1 - kTop > m[1] ? n1 - kTop : m[1];
                const float f0 = m[0] == n0 ? 1.f : ex2(m[0] - n0), f1 = m[1] == n1 ? 1.f : ex2(m[1] - n1);
                m[0] = n0; m[1] = n1;
                l[0] *= f0; l[1] *= f1;
#pragma unroll
                for (int i = 0; i < MT; ++i) { o[i][0] *= f0; o[i][1] *= f1; o[i][2] *= f0; o[i][3] *= f1; }
            }
            const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
            const bool plain = st[0].plain & st[1].plain;
            uint32_t p[2][2];
            float back[2][2];             // not plain: what the products of 16 tokens and their sums of weights are multiplied by
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                s[x][0] -= m0; s[x][1] -= m1; s[x][2] -= m0; s[x][3] -= m1;
                float w0 = __uint_as_float((uint32_t)(127 - (int)st[x].ve) << 23), w1 = w0;
                if (!plain) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(s[x][i], s[x][i + 2]);
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        // a whole number of powers of two; 16 tokens that weigh less than 2^-120 of the run's product may go
                        const float up = fminf(fmaxf(floorf(kTop - top), -kLazyMax), 120.f);
                        s[x][i] += up;
                        s[x][i + 2] += up;
                        back[x][i] = __uint_as_float((uint32_t)(127 - (int)up) << 23);
                    }
                    w0 *= back[x][0];
                    w1 *= back[x][1];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[x][i] = ex2(s[x][i]);
                l[0] = fmaf(s[x][0] + s[x][2], w0, l[0]);
                l[1] = fmaf(s[x][1] + s[x][3], w1, l[1]);
                p[x][0] = transpose8x8(pack_half(s[x][0], s[x][1]));
                p[x][1] = transpose8x8(pack_half(s[x][2], s[x][3]));
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int w = 0; w < HD / 32; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t y = __byte_perm(v[x][0][w], v[x][1][w], h ? 0x7362 : 0x5140), z = __byte_perm(v[x][2][w], v[x][3][w], h ? 0x7362 : 0x5140);
                        if (plain) {
                            mma16(o[2 * w + h], half_pair(y), half_pair_hi(y), half_pair(z), half_pair_hi(z), p[x][0], p[x][1]);
                        } else {
                            float d[4] = {};
                            mma16(d, half_pair(y), half_pair_hi(y), half_pair(z), half_pair_hi(z), p[x][0], p[x][1]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[2 * w + h][i] = fmaf(d[i], st[x].vr * back[x][i & 1], o[2 * w + h][i]);
                        }
                    }
        };
        for (int tok = tok0; tok < tok1; tok += R::kTokens, ++used) {
            const uint32_t st = used % NS;
            if (!__all_sync(0xffffffffu, mbar_wait(bar_at + 8 * st, (used / NS) & 1, ctl, kKernelPaged * 100 + 1))) {
                const long long t_end = clock64() + (1LL << 19);      // copies in flight land before shared memory is given back
                while (clock64() < t_end) __nanosleep(256);
                return;
            }
#pragma unroll
            for (int i = 0; i < NG; i += 2)
                if (tok + 16 * i < tok1) compute(tok + 16 * i, ring + st * R::kStage + i * 16 * HD, &granules[warp][st][i]);
            __syncwarp();
            if (tok + NS * R::kTokens < tok1) load(tok + NS * R::kTokens);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
            l[1] += __shfl_xor_sync(0xffffffffu, l[1], d);
        }
        if (u == begin && stop == end) {                 // all of the item
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = col0 + 2 * t + i;
                if (r >= rows) continue;
                const int n = r / a.group, h = head * a.group + r % a.group;
                const float f = l[i] == 0.f ? 0.f : 1.f / l[i];
                uint32_t *dst = reinterpret_cast<uint32_t *>(a.o + b * a.o_stride[0] + n * a.o_stride[1] + h * a.o_stride[2] + g * (HD / 8));
#pragma unroll
                for (int x = 0; x < MT; ++x) {
                    const __nv_bfloat162 y = __floats2bfloat162_rn(l[i] == 0.f ? 0.f : o[x][i] * f, l[i] == 0.f ? 0.f : o[x][i + 2] * f);
                    dst[x] = *reinterpret_cast<const uint32_t *>(&y);
                }
                if (a.lse && g == 0) a.lse[((long long)b * a.n_new + n) * a.n_q + h] = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * 0.6931471805599453f;
            }
        } else {
            const int slot = u == u_first ? 0 : 1;
            const long long at = ((long long)worker * 2 + slot) * kCols;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int cidx = 2 * t + i;
                if (col0 + cidx >= rows) continue;
                float2 *dst = reinterpret_cast<float2 *>(a.part + (at + cidx) * HD + g * (HD / 8));
#pragma unroll
                for (int x = 0; x < MT; ++x) dst[x] = make_float2(o[x][i], o[x][i + 2]);
                if (g == 0) a.ml[at + cidx] = make_float2(m[i], l[i]);
            }
        }
        if (stop == end && lane == 0) {
            const int w0 = u_first <= begin ? worker : deal.owner(begin);
            a.shared_by[(long long)b * per_seq + item] = make_int4(w0, worker, deal.first(w0) < begin ? 1 : 0, 0);
        }
        u = stop;
    }
}

// The parts of items that more than one worker had, added in the order of the tokens (each of a block's warps every
// fourth or sixteenth of them, then the warps' sums);
// and rows of sequences without tokens.  A block a row; a lane holds dims l, l + 32, ...
template <int HD, int kCombineWarps>
__global__ void __launch_bounds__(kCombineWarps * 32) paged_combine_kernel(const PagedArgs a) {
    constexpr int N = HD / 32;
    __shared__ float sum[kCombineWarps][HD], top[kCombineWarps], weights[kCombineWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = a.group * a.n_new;
    const int r = (int)(blockIdx.x % rows), head = (int)(blockIdx.x / rows % a.n_kv), b = (int)(blockIdx.x / rows / a.n_kv);
    const int n = r / a.group, h = head * a.group + r % a.group, col = r % kCols;
    const bool empty = length_of(a, b) == 0;
    griddep_wait();        // launched early, behind the kernel whose parts it adds
    int4 by = empty ? make_int4(0, 0, 0, 0) : a.shared_by[((long long)b * a.n_kv + head) * a.col_tiles + r / kCols];
    // (a warp that gave up on a wait has written nothing, neither here nor of its parts: what stands there may be anything)
    by = make_int4(min(max(by.x, 0), a.workers - 1), min(max(by.y, 0), a.workers - 1), by.z & 1, 0);
    if (!empty && by.x == by.y) return;
    float m = -INFINITY, l = 0.f;
    if (!empty) {
        // each warp its own maximum, some parts in flight
        constexpr int U = kCombineWarps == 4 ? 2 : 8;
        float o[N] = {};
        for (int w0 = by.x + warp; w0 <= by.y; w0 += U * kCombineWarps) {
            float2 ml[U];
            float v[U][N] = {};
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int w = w0 + i * kCombineWarps;
                ml[i] = make_float2(-INFINITY, 0.f);
                if (w <= by.y) {
                    const long long at = ((long long)w * 2 + (w == by.x ? by.z : 0)) * kCols + col;
                    ml[i] = a.ml[at];
#pragma unroll
                    for (int x = 0; x < N; ++x) v[i][x] = a.part[at * HD + x * 32 + lane];
                }
            }
            float now = m;
#pragma unroll
            for (int i = 0; i < U; ++i) now = fmaxf(now, ml[i].x);
            const float ref = now == -INFINITY ? 0.f : now, keep = ex2(m - ref);
            m = now;
            l *= keep;
#pragma unroll
            for (int x = 0; x < N; ++x) o[x] *= keep;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const float f = ex2(ml[i].x - ref);
                l = fmaf(ml[i].y, f, l);
#pragma unroll
                for (int x = 0; x < N; ++x) o[x] = fmaf(v[i][x], f, o[x]);
            }
        }
#pragma unroll
        for (int x = 0; x < N; ++x) sum[warp][x * 32 + lane] = o[x];
        if (lane == 0) {
            top[warp] = m;
            weights[warp] = l;
        }
        __syncthreads();
        m = top[0];
#pragma unroll
        for (int i = 1; i < kCombineWarps; ++i) m = fmaxf(m, top[i]);
        const float ref = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < kCombineWarps; ++i) l = fmaf(weights[i], ex2(top[i] - ref), l);
    }
    __nv_bfloat16 *dst = a.o + b * a.o_stride[0] + n * a.o_stride[1] + h * a.o_stride[2];
    const float f = l == 0.f ? 0.f : 1.f / l;
    for (int d = threadIdx.x; d < HD; d += kCombineWarps * 32) {
        float y = 0.f;
        if (!empty)
#pragma unroll
            for (int i = 0; i < kCombineWarps; ++i) y = fmaf(sum[i][d], ex2(top[i] - (m == -INFINITY ? 0.f : m)), y);
        dst[d] = __float2bfloat16(l == 0.f ? 0.f : y * f);
    }
    if (a.lse && threadIdx.x == 0) a.lse[((long long)b * a.n_new + n) * a.n_q + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

int workers_for(int num_sms, int hd) { return num_sms * kWarps * (hd == 64 ? Ring<64>::kBlocks : hd == 96 ? Ring<96>::kBlocks : Ring<128>::kBlocks); }

}  // namespace

int col_tiles_of(const flashmhf_paged_attention_params &p) { return (p.n_q / p.pages.n_kv * p.n_new + kCols - 1) / kCols; }

size_t paged_attention_workspace_bytes(const flashmhf_paged_attention_params &p) {
    return (size_t)workers_for(num_sms(), p.pages.head_dim) * 2 * kCols * (p.pages.head_dim + 2) * sizeof(float) +
           (size_t)p.seq.B * p.pages.n_kv * col_tiles_of(p) * sizeof(int4);
}

int paged_attention(const flashmhf_paged_attention_params &p, const DeviceCtl &ctl, cudaStream_t st, int *n_launch) {
    PagedArgs a{};
    const flashmhf_kv_pages &g = p.pages;
    a.k = static_cast<const uint8_t *>(g.k); a.v = static_cast<const uint8_t *>(g.v);
    a.k_scale = g.k_scale; a.v_scale = g.v_scale; a.page_stride = g.page_stride;
    a.lengths = p.seq.lengths; a.table = p.seq.table; a.table_stride = p.seq.table_stride;
    a.q = static_cast<const __nv_bfloat16 *>(p.q); a.o = static_cast<__nv_bfloat16 *>(p.o);
    for (int i = 0; i < 3; ++i) { a.q_stride[i] = p.q_stride[i]; a.o_stride[i] = p.o_stride[i]; }
    a.lse = p.lse; a.index = ctl.index;
    a.B = p.seq.B; a.max_pages = p.seq.max_pages; a.num_pages = g.num_pages; a.n_kv = g.n_kv; a.n_q = p.n_q; a.n_new = p.n_new;
    a.log_page = g.page_size == 16 ? 4 : g.page_size == 32 ? 5 : g.page_size == 64 ? 6 : 7;
    a.group = p.n_q / g.n_kv;
    a.col_tiles = col_tiles_of(p);
    a.workers = workers_for(ctl.num_sms, g.head_dim);
    a.part = static_cast<float *>(p.workspace);
    a.ml = reinterpret_cast<float2 *>(a.part + (size_t)a.workers * 2 * kCols * g.head_dim);
    a.shared_by = reinterpret_cast<int4 *>(a.ml + (size_t)a.workers * 2 * kCols);
    a.c = p.scale * 1.4426950408889634f;
    const long long rows = (long long)a.B * a.n_new * a.n_q;
    if (rows > 0x7fffffffll) return FLASHMHF_ERR_BAD_SHAPE;
    a.wait = wait_args(&ctl);
    auto kernel = g.head_dim == 64 ? paged_attention_kernel<64> : g.head_dim == 96 ? paged_attention_kernel<96> : paged_attention_kernel<128>;
    // An item has workers / items parts where its sequence is as long as the others, and up to all of them where it is the only long one.
    // With few items there are few rows as well, and a block of 16 warps for each costs nothing: two of 65537 tokens, over 200 parts
    // an item, 53 us by four warps, 39 by sixteen; 64 of 8192, about four parts, 183 and 212.
    const bool wide = (long long)a.B * g.n_kv * a.col_tiles * 16 <= a.workers;
    auto combine = g.head_dim == 64   ? (wide ? paged_combine_kernel<64, 16> : paged_combine_kernel<64, 4>)
                   : g.head_dim == 96 ? (wide ? paged_combine_kernel<96, 16> : paged_combine_kernel<96, 4>)
                                      : (wide ? paged_combine_kernel<128, 16> : paged_combine_kernel<128, 4>);
    const size_t smem = (size_t)kWarps * (g.head_dim == 64 ? Ring<64>::kBytes : g.head_dim == 96 ? Ring<96>::kBytes : Ring<128>::kBytes);
    cudaError_t e = cudaSuccess;
    static std::atomic<bool> done[3][64];      // the attribute is per kernel and device
    std::atomic<bool> &set = done[g.head_dim / 32 - 2][ctl.device];
    if (!set.load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        set.store(e == cudaSuccess, std::memory_order_release);
    }
    if (e == cudaSuccess) e = launch_kernel(false, kernel, dim3((unsigned)(a.workers / kWarps)), dim3(kWarps * 32), smem, st, a);
    if (e == cudaSuccess) e = launch_kernel(true, combine, dim3((unsigned)rows), dim3((wide ? 16 : 4) * 32), 0, st, a);
    if (e != cudaSuccess) {
        set_cuda_error(e, "paged attention launch");
        return FLASHMHF_ERR_CUDA;
    }
    *n_launch += 2;
    return FLASHMHF_OK;
}

}  // namespace fmhf
