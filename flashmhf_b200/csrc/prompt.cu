// Attention over packed prompts, bf16, sm_100a:  O = softmax(scale Q K^T + mask) V  per sequence and query head.
//
// A work item is 256 consecutive rows of one sequence and query head, in two tiles of 128 rows; both read the same tiles of 64 keys.  Per tile
// of keys and tile of rows the tensor core computes S = Q K^T (128 x 64, fp32 in tensor memory), one warpgroup (a thread a row) takes the
// running maximum and P = bf16(2^(c s - c m)) and writes it over S, and the tensor core adds P V to O (fp32, in tensor memory over all
// keys): scores and weights never leave the SM.
//
// Bound: latencies first, exponentials second.  The special function units take 512 clk for 128 x 64 exponentials, the products 370 (a head of 64) to
// 650 clk (128); but from S to P a step is a chain of some 1800 clk (barriers, tensor memory both ways, the maximum, a warp's exponentials).
// So four chains are under way: each tile of rows has two buffers of S and two warpgroups, which take its steps in turn.  A step needs
// nothing of the one before but its maximum, which is known early and goes through shared memory.
//
// The maximum is lazy: O is multiplied by 2^(c m_old - c m_new) only where a new maximum is more than 2^8 above the one in use (P is then
// at most 256, and P, its sum and O are all in one scale), so that almost no step touches O.
//
// No product writes tensor memory that another one may still be reading on the strength of the order of issue alone (that order is promised for
// products of one accumulator and shape).  A head of 64 leaves room for P beside S; with heads of 96 and 128 P lies over S, and S of step s + 2
// waits until the product that reads P of step s is done.
//
// Work items are handed out by the hardware: the grid has a block for each, a resident block takes over one that has not started
// (clusterlaunchcontrol) while it works on its own.
//
// Warp roles: 0-15 softmax (tile of rows = warp / 8, parity of the steps = warp / 4 % 2, TMEM lane quarter = warp % 4), 16 work items and TMA, 17
// issues S of both tiles, 18 and 19 O += P V of one each; 18 also clears the rows of V behind the end of a sequence (a weight of 0 does not undo a
// NaN of the next one).
#include <atomic>

#include "paged.cuh"
#include "tc_common.cuh"
#include "tensormap.cuh"

namespace fmhf {
namespace {

constexpr int kRows = 128, kItemRows = 2 * kRows, kKeys = 64;
constexpr int kSoftmaxWarps = 16, kThreads = (kSoftmaxWarps + 4) * 32;
constexpr int kKernelPrompt = 6;                  // status codes 601..
constexpr float kLazy = 65536.f;                  // the sum of a row's weights of a step above which its reference is set anew
constexpr int kLag = 8;
constexpr int kMaxStages = 8;

template <int HD>
struct PromptCfg {
    static constexpr int kChunks = (HD + 63) / 64, kStages = HD == 64 ? 8 : 4, kQBufs = HD == 64 ? 2 : 1;
    static constexpr uint32_t kQChunk = kRows * 128, kKChunk = kKeys * 128;     // 64 columns of a tile
    static constexpr uint32_t kQTile = kChunks * kQChunk, kTile = kChunks * kKChunk;
    static constexpr uint32_t kOffQ = 0, kOffK = kQBufs * 2 * kQTile, kOffV = kOffK + kStages * kTile;
    static constexpr uint32_t kOffMsg = kOffV + kStages * kTile, kOffEnd = kOffMsg + 4 * kRows * 4;   // [tile][parity][row]: maxima; maxima and sums (of two items)
    static constexpr uint32_t kOffBar = kOffEnd + 2 * 4 * kRows * 8, kTotal = kOffBar + 1024 + 1024;
    // tensor memory: two buffers for S of either tile of rows, O of both, and P: over S, or by itself where there is room
    static constexpr bool kOverlay = HD != 64;
    static constexpr uint32_t kColP = kOverlay ? 0 : 256, kPStride = kOverlay ? kKeys : kKeys / 2, kColO = kOverlay ? 256 : 384, kOStride = HD == 64 ? 64 : 128;
};

// SFULL: S computed into a buffer; SFREE: it is in registers; PFULL: P written, O scaled if need be; PVDONE: the product that read P is done (tile
// t, buffer b: + 2 t + b); OFULL: the last one of an item; OFREE: O has been read out (+ t); MSG: the maximum that a step was taken with (tile t, quarter q,
// steps of parity b: + 8 t + 2 q + b); ITEM*: the ring of work items; NEXT: the answer to a request for one.
enum { PB_QFULL = 0, PB_QEMPTY = 2, PB_SFULL = 4, PB_PFULL = 8, PB_PVDONE = 12, PB_OFULL = 16, PB_OFREE = 18, PB_ITEMFULL = 20, PB_ITEMEMPTY = 22,
       PB_NEXT = 24, PB_MSG = 25, PB_SFREE = 41, PB_KFULL = 45, PB_KEMPTY = PB_KFULL + kMaxStages, PB_VFULL = PB_KEMPTY + kMaxStages,
       PB_VEMPTY = PB_VFULL + kMaxStages, PB_VRAW = PB_VEMPTY + kMaxStages, PB_COUNT = PB_VRAW + kMaxStages };
constexpr uint32_t kOffNext = (PB_COUNT * 8 + 15) / 16 * 16, kOffItems = kOffNext + 16, kOffCtl = kOffItems + 2 * 48;
static_assert(kOffCtl + 8 <= 1024, "control area");

struct PromptItem {
    int q0, lq;          // first row of the item in the packed rows; rows of the sequence from there on
    int k0, lk;          // first key and keys of the sequence
    int see;             // keys that the item's first row sees, before clamping: row r sees min(lk, see + r) (causal) or lk
    int n0, n1;          // tiles of keys for the two tiles of rows
    int head;            // -1: no more items
};

struct PromptArgs {
    __nv_bfloat16 *o;
    long long o_tok, o_head;
    float *lse;
    const int32_t *cu_q, *cu_k;
    int B, tokens_q, tokens_k, n_q, group, causal, n_items;
    float c;             // |scale| log2(e), at least a tiny number (masked scores are -inf, and 0 times that is not a number)
    int negate;          // scale < 0
    WaitArgs wait;
};

// Item `index`: the last rows of each sequence, which see the most keys when the call is causal, come first.  Sequence b owns the slots
// from cu[b] / 256 + b on, at least as many as it has items.
__device__ __forceinline__ bool prompt_item(const PromptArgs &a, int index, PromptItem &w) {
    const int slots = a.tokens_q / kItemRows + a.B, slot = slots - 1 - index / a.n_q;
    w.head = index % a.n_q;
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(a.cu_q + mid) / kItemRows + mid <= slot) lo = mid;
        else hi = mid - 1;
    }
    const int q0 = __ldg(a.cu_q + lo), q1 = __ldg(a.cu_q + lo + 1), k0 = __ldg(a.cu_k + lo), k1 = __ldg(a.cu_k + lo + 1);
    if (q0 < 0 || q1 > a.tokens_q || q1 < q0 || k0 < 0 || k1 > a.tokens_k || k1 < k0) {
        note_index(a.wait.status, kPromptRows);
        return false;
    }
    const int r0 = (slot - (q0 / kItemRows + lo)) * kItemRows, lq = q1 - q0, lk = k1 - k0;
    if (r0 < 0 || r0 >= lq) return false;
    w.q0 = q0 + r0;
    w.lq = lq - r0;
    w.k0 = k0;
    w.lk = lk;
    w.see = a.causal ? r0 + 1 + lk - lq : lk;
    auto tiles = [&](int first, int rows) {      // tiles of keys that rows first .. first + rows - 1 need
        rows = min(rows, w.lq - first);
        if (rows <= 0) return 0;
        const int most = a.causal ? min(lk, max(0, w.see + first + rows - 1)) : lk;
        return (most + kKeys - 1) / kKeys;
    };
    w.n0 = tiles(0, kRows);
    w.n1 = tiles(kRows, kRows);
    return true;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// 2^x of both halves on the FMA pipe: x = n + f, n whole, |f| <= 1/2 (adding 1.5 * 2^23 rounds x to n and leaves it in the low bits), and a cubic in f of
// relative error 7.5e-5 at most, a fiftieth of the rounding of P to bf16 (fitted here: least squares in the relative error, reweighted
// until its extremes were level).  Below 2^-126 the result is 2^-126 or so, not 0: nothing beside a largest P of 1, but a row that
// sees nothing has to be known by its maximum.  What is not a number becomes so large that no finite result is left.
__device__ __forceinline__ f32x2 f2_exp2(f32x2 x) {
    float a, b, u, v;
    f2_unpack(x, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-126.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-126.f));
    x = f2_pack(a, b);
    const f32x2 magic = f2_pack(12582912.f, 12582912.f), back = f2_pack(-12582912.f, -12582912.f), minus = f2_pack(-1.f, -1.f);
    const f32x2 r = f2_add(x, magic), f = f2_fma(f2_add(r, back), minus, x);
    f32x2 y = f2_fma(f2_pack(0.0551716685f, 0.0551716685f), f, f2_pack(0.242611125f, 0.242611125f));
    y = f2_fma(y, f, f2_pack(0.693260968f, 0.693260968f));
    y = f2_fma(y, f, f2_pack(0.999928057f, 0.999928057f));
    f2_unpack(r, a, b);
    f2_unpack(y, u, v);
    return f2_pack(__int_as_float(__float_as_int(u) + (__float_as_int(a) << 23)), __int_as_float(__float_as_int(v) + (__float_as_int(b) << 23)));
}

// Bounded waits, in line: a call would spill what a softmax thread holds.  Of one thread; and of a whole warp, with the same answer for all lanes
// (those of a warp that gives up leave its loop together).
__device__ __forceinline__ bool thread_wait(uint32_t bar, uint32_t parity, const WaitCtl &ctl, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (*ctl.abort) return false;
        if (clock64() - t0 > ctl.g.limit_cycles) {
            *ctl.abort = 1;
            atomicCAS(ctl.g.status, 0, code);
            atomicExch(ctl.g.abort_seq, ctl.g.seq);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const WaitCtl &ctl, int code) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const long long t0 = clock64();
    while (true) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if (__any_sync(0xffffffffu, *ctl.abort)) return false;
        if (__any_sync(0xffffffffu, clock64() - t0 > ctl.g.limit_cycles)) {
            *ctl.abort = 1;
            atomicCAS(ctl.g.status, 0, code);
            atomicExch(ctl.g.abort_seq, ctl.g.seq);
            return false;
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const PromptArgs args) {
    using L = PromptCfg<HD>;
    constexpr int NS = L::kStages, NQ = L::kQBufs;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *gbase = smem_raw + (base - raw);
    const uint32_t sQ = base + L::kOffQ, sK = base + L::kOffK, sV = base + L::kOffV, sBar = base + L::kOffBar;
    volatile int *items = reinterpret_cast<volatile int *>(gbase + L::kOffBar + kOffItems);
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gbase + L::kOffBar + kOffCtl);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(gbase + L::kOffBar + kOffCtl + 4);
    auto bar = [&](int i) { return sBar + 8u * i; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtl ctl{abort_flag, args.wait};
    constexpr int W = kKernelPrompt * 100, kLoad = kSoftmaxWarps, kIssue = kLoad + 1;

    if (threadIdx.x == 0) {
        *abort_flag = launch_aborted(args.wait);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(PB_QFULL + i), 1);
            mbar_init(bar(PB_QEMPTY + i), 1);
            mbar_init(bar(PB_OFULL + i), 1);
            mbar_init(bar(PB_OFREE + i), 8);
            mbar_init(bar(PB_ITEMFULL + i), 1);
            mbar_init(bar(PB_ITEMEMPTY + i), kSoftmaxWarps + 3);      // every warp but the one that fills it
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(PB_SFULL + i), 1);
            mbar_init(bar(PB_PFULL + i), 4);
            mbar_init(bar(PB_SFREE + i), 4);
            mbar_init(bar(PB_PVDONE + i), 1);
        }
        for (int i = 0; i < 16; ++i) mbar_init(bar(PB_MSG + i), 1);
        mbar_init(bar(PB_NEXT), 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(bar(PB_KFULL + i), 1);
            mbar_init(bar(PB_KEMPTY + i), 1);
            mbar_init(bar(PB_VFULL + i), 1);
            mbar_init(bar(PB_VEMPTY + i), 2);
            mbar_init(bar(PB_VRAW + i), 1);
        }
        fence_mbar_init();
    }
    if (warp == kIssue) tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Work item `seq` of this block, after a wait for it.
    auto read_item = [&](int seq, PromptItem &w) {
        volatile int *p = items + (seq & 1) * 12;
        w.q0 = p[0]; w.lq = p[1]; w.k0 = p[2]; w.lk = p[3]; w.see = p[4]; w.n0 = p[5]; w.n1 = p[6]; w.head = p[7];
    };
    auto next_item = [&](int seq, PromptItem &w) -> bool {       // for a whole warp; false: no more, or given up
        if (!warp_wait(bar(PB_ITEMFULL + (seq & 1)), (seq >> 1) & 1, ctl, W + 1)) return false;
        read_item(seq, w);
        warp_arrive(bar(PB_ITEMEMPTY + (seq & 1)));
        return w.head >= 0;
    };

    if (*abort_flag) {
        // nothing: fall through to the teardown
    } else if (warp >= kSoftmaxWarps) {
        // A softmax thread holds a row of S: 512 x 104 + 128 x 56 registers of the 640 x 96 that the launch has.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == kLoad) {
            // -------------------------------------------------------------- work items and TMA
            if (lane == 0) {
                tma_prefetch_desc(&tmQ);
                tma_prefetch_desc(&tmK);
                tma_prefetch_desc(&tmV);
                int seq = 0, n_q = 0, asked = 0;
                uint32_t g = 0;          // tiles of keys so far
                bool ok = true;
                int index = blockIdx.x;
                const uint32_t answer = sBar + kOffNext;
                while (ok) {
                    // ask for the item after this one: the answer comes while this one is worked on
                    if (index >= 0) {
                        mbar_arrive_expect_tx(bar(PB_NEXT), 16);
                        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
                                     "r"(bar(PB_NEXT))
                                     : "memory");
                    }
                    PromptItem w{};
                    w.head = -1;
                    if (index < 0 || prompt_item(args, index, w)) {
                        const int s = seq & 1;
                        if (seq >= 2 && !thread_wait(bar(PB_ITEMEMPTY + s), ((seq >> 1) - 1) & 1, ctl, W + 2)) break;
                        volatile int *p = items + s * 12;
                        p[0] = w.q0; p[1] = w.lq; p[2] = w.k0; p[3] = w.lk; p[4] = w.see; p[5] = w.n0; p[6] = w.n1; p[7] = w.head;
                        mbar_arrive(bar(PB_ITEMFULL + s));
                        ++seq;
                    }
                    if (index < 0) break;
                    const int n = w.head < 0 ? 0 : max(w.n0, w.n1);
                    if (n > 0) {
                        const int qb = n_q % NQ;
                        if (n_q >= NQ && !thread_wait(bar(PB_QEMPTY + qb), (n_q / NQ - 1) & 1, ctl, W + 3)) break;
                        ++n_q;
                        mbar_arrive_expect_tx(bar(PB_QFULL + qb), ((w.n0 > 0) + (w.n1 > 0)) * L::kQTile);
                        for (int t = 0; t < 2; ++t)
                            for (int c = 0; c < ((t ? w.n1 : w.n0) > 0 ? L::kChunks : 0); ++c)
                                tma_load_3d(sQ + (qb * 2 + t) * L::kQTile + c * L::kQChunk, &tmQ, bar(PB_QFULL + qb), c * 64, w.head, w.q0 + t * kRows);
                    }
                    const int kh = w.head / args.group;
                    for (int j = 0; j < n; ++j, ++g) {
                        const uint32_t st = g % NS, lap = (g / NS) & 1;
                        if (!thread_wait(bar(PB_KEMPTY + st), lap ^ 1, ctl, W + 4)) { ok = false; break; }
                        mbar_arrive_expect_tx(bar(PB_KFULL + st), L::kTile);
                        for (int c = 0; c < L::kChunks; ++c)
                            tma_load_3d(sK + st * L::kTile + c * L::kKChunk, &tmK, bar(PB_KFULL + st), c * 64, kh, w.k0 + j * kKeys);
                        if (!thread_wait(bar(PB_VEMPTY + st), lap ^ 1, ctl, W + 5)) { ok = false; break; }
                        const uint32_t full = bar(((j + 1) * kKeys > w.lk ? PB_VRAW : PB_VFULL) + st);
                        mbar_arrive_expect_tx(full, L::kTile);
                        for (int c = 0; c < L::kChunks; ++c) tma_load_3d(sV + st * L::kTile + c * L::kKChunk, &tmV, full, c * 64, kh, w.k0 + j * kKeys);
                    }
                    if (!ok || !thread_wait(bar(PB_NEXT), asked++ & 1, ctl, W + 6)) break;
                    uint32_t got, next;
                    asm volatile(
                        "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\tld.shared.b128 h, [%2];\n\t"
                        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, h;\n\t}"
                        : "=r"(got), "=r"(next)
                        : "r"(answer)
                        : "memory");
                    fence_async_smem();          // the answer has been read before the next one is written there
                    index = got ? (int)next : -1;
                }
            }
        } else if (warp == kIssue) {
            // -------------------------------------------------------------- S of both tiles, whichever can go on
            if (lane == 0) {
                constexpr uint32_t idesc = umma_idesc(kRows, kKeys, false, false);
                const uint64_t dQ0 = desc_kmajor(sQ), dK0 = desc_kmajor(sK);
                PromptItem w;
                uint32_t g = 0, steps[2] = {0, 0};      // tiles of keys so far, of all items; those that the tiles of rows needed
                int n_q = 0;
                bool ok = true;
                for (int seq = 0; ok; ++seq) {
                    if (!thread_wait(bar(PB_ITEMFULL + (seq & 1)), (seq >> 1) & 1, ctl, W + 8)) break;
                    read_item(seq, w);
                    mbar_arrive(bar(PB_ITEMEMPTY + (seq & 1)));
                    if (w.head < 0) break;
                    const int n = max(w.n0, w.n1), need[2] = {w.n0, w.n1};
                    if (n == 0) continue;
                    const int qb = n_q % NQ;
                    if (!thread_wait(bar(PB_QFULL + qb), (n_q / NQ) & 1, ctl, W + 9)) break;
                    ++n_q;
                    int next[2] = {0, 0}, there = 0, back = 0;      // S issued; tiles of keys that have come, that were given back
                    long long t0 = 0;
                    while (back < n) {
                        bool went = false;
                        if (there < n && there <= max(next[0], next[1])) {
                            const uint32_t x = g + there;
                            if (mbar_test(bar(PB_KFULL + x % NS), (x / NS) & 1)) {
                                ++there;
                                went = true;
                            }
                        }
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            if (next[t] >= min(need[t], there)) continue;
                            const uint32_t st = (g + next[t]) % NS, s = steps[t] + next[t], b = s & 1;
                            // its buffer is free: S of two steps before is in registers, or over it P has been read
                            if (s >= 2 && !mbar_test(bar((L::kOverlay ? PB_PVDONE : PB_SFREE) + t * 2 + b), ((s >> 1) - 1) & 1)) continue;
                            tc_fence_after();
#pragma unroll
                            for (int k = 0; k < HD / 16; ++k)
                                umma_ss(tmem + (t * 2 + b) * kKeys, dQ0 + (((qb * 2 + t) * L::kQTile + (k >> 2) * L::kQChunk + (k & 3) * 32) >> 4),
                                        dK0 + ((st * L::kTile + (k >> 2) * L::kKChunk + (k & 3) * 32) >> 4), idesc, k > 0 ? 1u : 0u);
                            umma_commit(bar(PB_SFULL + t * 2 + b));
                            ++next[t];
                            went = true;
                        }
                        while (back < there && next[0] >= min(need[0], back + 1) && next[1] >= min(need[1], back + 1)) {
                            umma_commit(bar(PB_KEMPTY + (g + back) % NS));
                            if (++back == n) umma_commit(bar(PB_QEMPTY + qb));
                        }
                        if (went) t0 = 0;
                        else if (t0 == 0) t0 = clock64();
                        else if (*abort_flag) { ok = false; break; }
                        else if (clock64() - t0 > args.wait.limit_cycles) {
                            *abort_flag = 1;
                            atomicCAS(args.wait.status, 0, W + 10);
                            atomicExch(args.wait.abort_seq, args.wait.seq);
                            ok = false;
                            break;
                        }
                    }
                    g += n;
                    steps[0] += w.n0;
                    steps[1] += w.n1;
                }
            }
        } else {
            // -------------------------------------------------------------- O += P V of one tile of rows
            const int t = warp - kIssue - 1;
            constexpr uint32_t idesc = umma_idesc(kRows, HD, false, true);
            const uint64_t dV0 = desc_mnmajor(sV, L::kKChunk);
            const uint32_t tP = tmem + L::kColP + t * 2 * L::kPStride, tO = tmem + L::kColO + t * L::kOStride;
            PromptItem w;
            uint32_t g = 0, steps = 0, seen = 0;      // (seen: parities of the stages' raw barriers, which only tiles with the end of a sequence use)
            int outs = 0;
            bool ok = true;
            for (int seq = 0; ok && next_item(seq, w); ++seq) {
                const int n = max(w.n0, w.n1), mine = t ? w.n1 : w.n0;
                for (int j = 0; j < n; ++j) {
                    const uint32_t st = (g + j) % NS, lap = ((g + j) / NS) & 1, s = steps + j, b = s & 1;
                    if (t == 0 && (j + 1) * kKeys > w.lk) {
                        if (!warp_wait(bar(PB_VRAW + st), seen >> st & 1, ctl, W + 7)) { ok = false; break; }
                        seen ^= 1u << st;
                        for (int i = (w.lk - j * kKeys) * 8 + lane; i < kKeys * 8; i += 32)
#pragma unroll
                            for (int c = 0; c < L::kChunks; ++c) st_shared_v4(sV + st * L::kTile + c * L::kKChunk + i * 16, 0, 0, 0, 0);
                        fence_async_smem();
                        warp_arrive(bar(PB_VFULL + st));
                    }
                    if (!warp_wait(bar(PB_VFULL + st), lap, ctl, W + 11)) { ok = false; break; }
                    if (j >= mine) {       // the other tile of rows goes on alone: every phase is still seen, and every stage given back
                        if (lane == 0) mbar_arrive(bar(PB_VEMPTY + st));
                        continue;
                    }
                    if (j == 0 && outs > 0 && !warp_wait(bar(PB_OFREE + t), (outs - 1) & 1, ctl, W + 12)) { ok = false; break; }
                    if (!warp_wait(bar(PB_PFULL + t * 2 + b), (s >> 1) & 1, ctl, W + 13)) { ok = false; break; }
                    tc_fence_after();
                    if (lane == 0) {
#pragma unroll
                        for (int k = 0; k < kKeys / 16; ++k)
                            umma_ts(tO, tP + b * L::kPStride + k * 8, dV0 + st * (L::kTile >> 4) + k * 128, idesc, (j > 0 || k > 0) ? 1u : 0u);
                        umma_commit(bar(PB_PVDONE + t * 2 + b));
                        umma_commit(bar(PB_VEMPTY + st));
                        if (j + 1 == mine) umma_commit(bar(PB_OFULL + t));
                    }
                    __syncwarp();
                }
                g += n;
                steps += mine;
                outs += mine > 0;
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax and output, a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        constexpr int NO = HD / 2;                   // columns of O that each of the two warpgroups of a tile writes out
        const int t = warp >> 3, par = (warp >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t tS = lanes + (t * 2 + par) * kKeys, tP = lanes + L::kColP + (t * 2 + par) * L::kPStride, tO = lanes + L::kColO + t * L::kOStride;
        const uint32_t msg_out = bar(PB_MSG + 8 * t + 2 * quarter + par), msg_in = bar(PB_MSG + 8 * t + 2 * quarter + (par ^ 1));
        volatile float *maxima = reinterpret_cast<volatile float *>(gbase + L::kOffMsg) + t * 2 * kRows + row;
        volatile float2 *ends = reinterpret_cast<volatile float2 *>(gbase + L::kOffEnd) + t * 2 * kRows + row;
        const int pair_bar = 1 + (t * 4 + quarter);
        const float c = args.c;
        PromptItem w;
        uint32_t steps = 0;
        int outs = 0;
        bool ok = true;
        for (int seq = 0; ok && (ok = next_item(seq, w)); ++seq) {
            const int mine = t ? w.n1 : w.n0, r = t * kRows + row;
            const int see = args.causal ? max(0, min(w.lk, w.see + r)) : w.lk;      // keys that this row sees
            const int all = __shfl_sync(0xffffffffu, see, 0);                       // ... and every row of this warp
            float m = -INFINITY, l = 0.f;      // the reference that this warpgroup's last step was taken with, and its weights' sum
            for (int j = (steps & 1) ^ par; j < mine; j += 2) {
                const uint32_t step = steps + j;
                if (!warp_wait(bar(PB_SFULL + t * 2 + par), (step >> 1) & 1, ctl, W + 15)) { ok = false; break; }
                tc_fence_after();
                // The product that read what P overwrites is done (over S that is so, or S could not have been computed).  Before the message:
                // whoever has that knows which phase of this barrier comes next.
                if (!L::kOverlay && step > 1) {
                    if (!warp_wait(bar(PB_PVDONE + t * 2 + par), ((step >> 1) - 1) & 1, ctl, W + 14)) { ok = false; break; }
                    tc_fence_after();
                }
                // what the step before was taken with; every message is waited for before the next one is sent
                bool heard = step == 0;
                float ref = m;
                auto hear = [&]() -> bool {
                    heard = true;
                    return warp_wait(msg_in, ((step - 1) >> 1) & 1, ctl, W + 16);
                };
                auto send = [&] {
                    maxima[par * kRows] = ref;
                    warp_arrive(msg_out);
                };
                if (j == 1) {
                    if (!hear()) { ok = false; break; }
                    ref = maxima[(par ^ 1) * kRows];
                }
                bool with_max = j == 0;
                float before = ref, sum;
                uint32_t p[32];
                while (true) {
                    float s[kKeys];
                    tmem_ld32x2_sync(tS, tS + 32, reinterpret_cast<uint32_t *>(s), reinterpret_cast<uint32_t *>(s) + 32);
                    if (args.negate)
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) s[i] = -s[i];
                    if ((j + 1) * kKeys > all) {
                        const int left = see - j * kKeys;
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) s[i] = i < left ? s[i] : -INFINITY;
                    }
                    if (with_max) {
                        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (int i = 4; i < kKeys; i += 8)
#pragma unroll
                            for (int k = 0; k < 4; ++k) top[k] = i + 4 < kKeys ? max3(top[k], s[i + k], s[i + 4 + k]) : fmaxf(top[k], s[i + k]);
                        before = ref;
                        ref = fmaxf(ref, fmaxf(max3(top[0], top[1], top[2]), top[3]));
                        if (!heard && !hear()) { ok = false; break; }
                        send();          // (no weight of this pass is above 1: it stays)
                    }
                    const float mc = ref == -INFINITY ? 0.f : -ref * c;
                    const f32x2 c2 = f2_pack(c, c), mc2 = f2_pack(mc, mc);
                    f32x2 sum0 = 0, sum1 = 0;
#pragma unroll
                    for (int i = 0; i < kKeys + kLag; i += 8) {
                        if (i < kKeys) {
#pragma unroll
                            for (int k = 0; k < 8; k += 2) {
                                f2_unpack(f2_fma(f2_pack(s[i + k], s[i + k + 1]), c2, mc2), s[i + k], s[i + k + 1]);
                                s[i + k] = ex2(s[i + k]);
                                s[i + k + 1] = ex2(s[i + k + 1]);
                            }
                        }
                        if (i >= kLag) {
                            const int y = i - kLag;
#pragma unroll
                            for (int k = 0; k < 8; k += 4) {
                                sum0 = f2_add(sum0, f2_pack(s[y + k], s[y + k + 1]));
                                sum1 = f2_add(sum1, f2_pack(s[y + k + 2], s[y + k + 3]));
                                p[(y + k) / 2] = pack_bf16(s[y + k], s[y + k + 1]);
                                p[(y + k) / 2 + 1] = pack_bf16(s[y + k + 2], s[y + k + 3]);
                            }
                        }
                    }
                    float a0, a1;
                    f2_unpack(f2_add(sum0, sum1), a0, a1);
                    sum = a0 + a1;
                    if (with_max) break;
                    bool stale = false;
                    if (!heard) {
                        if (!hear()) { ok = false; break; }
                        const float now = maxima[(par ^ 1) * kRows];
                        stale = now != ref;
                        ref = now;
                    }
                    if (__any_sync(0xffffffffu, stale)) continue;       // the other warpgroup took a new reference: once more with that
                    with_max = __any_sync(0xffffffffu, sum > kLazy || (ref == -INFINITY && sum > 0.f));
                    if (!with_max) {
                        send();
                        break;
                    }
                }
                if (!ok) break;
                if (!L::kOverlay) {
                    tc_fence_before();
                    warp_arrive(bar(PB_SFREE + t * 2 + par));
                }
                if (with_max && j > 0) {
                    if (!warp_wait(bar(PB_PVDONE + t * 2 + (par ^ 1)), ((step - 1) >> 1) & 1, ctl, W + 17)) { ok = false; break; }
                    tc_fence_after();
                    const float keep = before == ref ? 1.f : before == -INFINITY ? 0.f : ex2((before - ref) * c);
#pragma unroll
                    for (int d = 0; d < HD; d += 16) {
                        uint32_t o[16];
                        tmem_ld16_sync(tO + d, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                        tmem_st16(tO + d, o);
                    }
                }
                tmem_st32(tP, p);
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(bar(PB_PFULL + t * 2 + par));
                l = fmaf(l, m == ref ? 1.f : m == -INFINITY ? 0.f : ex2((m - ref) * c), sum);
                m = ref;
            }
            steps += mine;
            if (!ok) break;
            // maxima and sums of both warpgroups: the larger maximum is the later one
            volatile float2 *e = ends + (seq & 1) * 4 * kRows;
            e[par * kRows].x = m;
            e[par * kRows].y = l;
            named_bar_sync(pair_bar, 64);
            if (*abort_flag) { ok = false; break; }      // (set before a warp that gives up arrives here for the last time, below)
            const float m2 = e[(par ^ 1) * kRows].x, l2 = e[(par ^ 1) * kRows].y, top = fmaxf(m, m2);
            const float ref = top == -INFINITY ? 0.f : top;
            l = l * ex2((m - ref) * c) + l2 * ex2((m2 - ref) * c);
            if (mine > 0) {
                if (!(ok = warp_wait(bar(PB_OFULL + t), outs++ & 1, ctl, W + 18))) break;
                tc_fence_after();
            }
            const bool none = top == -INFINITY && l < 1e-20f;      // (l is not a number, or not finite, where a score is not a number)
            const float inv = 1.f / l;
            const bool mine_row = r < w.lq;
            __nv_bfloat16 *dst = args.o + (long long)(w.q0 + r) * args.o_tok + (long long)w.head * args.o_head + par * NO;
#pragma unroll
            for (int d = 0; d < NO; d += 16) {
                uint32_t o[16] = {};
                if (mine > 0) tmem_ld16_sync(tO + par * NO + d, o);
                if (mine_row)
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        uint32_t v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            v[k] = none ? 0u : pack_bf16(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
                        *reinterpret_cast<uint4 *>(dst + d + i) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
            }
            if (mine > 0) {
                tc_fence_before();
                warp_arrive(bar(PB_OFREE + t));
            }
            if (args.lse && mine_row && par == 0)
                args.lse[(long long)(w.q0 + r) * args.n_q + w.head] = none ? -INFINITY : (top * c + log2f(l)) * 0.6931471805599453f;
        }
        // (the warp with the other steps must not wait for this one; if this one gave up, it gives up at its next wait)
        asm volatile("bar.arrive %0, 64;" ::"r"(pair_bar) : "memory");
    }
    __syncwarp();
    if (*abort_flag) {
        // a wait ran out somewhere in this CTA: give copies and MMAs still in flight time to land before shared and tensor memory
        // are released
        const long long t_end = clock64() + (1LL << 19);
        while (clock64() < t_end) __nanosleep(256);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kIssue) tmem_dealloc(tmem, 512);
}

template <int HD>
int launch_prompt(const flashmhf_prompt_attention_params &p, const PromptArgs &a, int device, cudaStream_t st, int *n_launch) {
    CUtensorMap q, k, v;
    auto map = [&](CUtensorMap *m, const void *ptr, const int64_t *stride, int heads, int tokens, int rows) {
        if (tokens == 0) heads = tokens = 1;      // no keys at all: nothing is read through the map
        const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)heads, (uint64_t)tokens};
        const int64_t str[2] = {stride[1], stride[0]};
        const uint32_t box[3] = {64, 1, (uint32_t)rows};
        return encode_bf16_map(m, ptr, 3, dims, str, box);
    };
    int rc = map(&q, p.q, p.q_stride, p.n_q, p.tokens_q, kRows);
    if (rc == FLASHMHF_OK) rc = map(&k, p.k, p.k_stride, p.n_kv, p.tokens_k, kKeys);
    if (rc == FLASHMHF_OK) rc = map(&v, p.v, p.v_stride, p.n_kv, p.tokens_k, kKeys);
    if (rc != FLASHMHF_OK) return rc;
    const size_t smem = PromptCfg<HD>::kTotal;
    cudaError_t e = cudaSuccess;
    static std::atomic<bool> done[64];      // the attribute is per kernel and device
    if (!done[device].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(prompt_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        done[device].store(e == cudaSuccess, std::memory_order_release);
    }
    if (e == cudaSuccess) e = launch_kernel(false, prompt_attention_kernel<HD>, dim3((unsigned)a.n_items), dim3(kThreads), smem, st, q, k, v, a);
    if (e != cudaSuccess) {
        set_cuda_error(e, "prompt attention launch");
        return FLASHMHF_ERR_CUDA;
    }
    ++*n_launch;
    return FLASHMHF_OK;
}

}  // namespace

int prompt_attention(const flashmhf_prompt_attention_params &p, const DeviceCtl &ctl, cudaStream_t st, int *n_launch) {
    PromptArgs a{};
    a.o = static_cast<__nv_bfloat16 *>(p.o);
    a.o_tok = p.o_stride[0]; a.o_head = p.o_stride[1];
    a.lse = p.lse; a.cu_q = p.cu_q; a.cu_k = p.cu_k;
    a.B = p.B; a.tokens_q = p.tokens_q; a.tokens_k = p.tokens_k; a.n_q = p.n_q; a.group = p.n_q / p.n_kv; a.causal = p.causal != 0;
    const long long items = ((long long)p.tokens_q / kItemRows + p.B) * p.n_q;
    if (items > 0x3fffffffll) return FLASHMHF_ERR_BAD_SHAPE;
    a.n_items = (int)items;
    a.negate = p.scale < 0.f;
    const float c = (p.scale < 0.f ? -p.scale : p.scale) * 1.4426950408889634f;
    a.c = c > 1e-30f ? c : 1e-30f;
    a.wait = wait_args(&ctl);
    switch (p.head_dim) {
        case 64: return launch_prompt<64>(p, a, ctl.device, st, n_launch);
        case 96: return launch_prompt<96>(p, a, ctl.device, st, n_launch);
        default: return launch_prompt<128>(p, a, ctl.device, st, n_launch);
    }
}

}  // namespace fmhf
