// Attention over packed prompts, bf16, sm_100a:  O = softmax(scale Q K^T + mask) V  per sequence and query head.
//
// A work item is 256 consecutive rows of one sequence and query head, in two tiles of 128 rows; both read the same tiles of 128 keys.
// Per tile of keys and tile of rows the tensor core computes S = Q K^T (128 x 128, fp32 in tensor memory), one warpgroup (a thread a
// row) takes the running maximum and P = bf16(2^(c s - c m)) and puts it into tensor memory, and the tensor core adds P V to O (fp32, in
// tensor memory over all keys): scores and weights never leave the SM.
//
// Bound: the exponentials.  128 x 128 of them take the SM's special function units 1024 clk; the two products take 2 x 258 clk at a head of 64 and
// 2 x 516 at 128.  So the two tiles of an item are worked on by two warpgroups that take turns: while one does its arithmetic, the tensor
// core works for the other.
//
// The maximum is lazy: O is multiplied by 2^(c m_old - c m_new) only where a new maximum is more than 2^8 above the one in use (P is then
// at most 256, and P, its sum and O are all in one scale), so that almost no tile touches O.
//
// Tensor memory (512 columns).  A head of 64: S of the two tiles, P of the two (64 columns each), O of the two (64 each); the next S
// may be computed as soon as this one is in registers.  Heads of 96 and 128: O needs 2 x 128, so P lies over S, and the next S waits until
// the product that reads P is done (the order of issue would do, but is promised only for products of one accumulator and shape).
//
// Warp roles: 0-3 and 4-7 softmax of the two tiles (warp % 4 = TMEM lane quarter = 32 rows), 8 work items and TMA, 9 and 10 MMA issuers of
// the two tiles.  Warp 9 also clears the rows of V behind the end of a sequence (a weight of 0 does not undo a NaN of the next one).
#include <atomic>

#include "paged.cuh"
#include "tc_common.cuh"
#include "tensormap.cuh"

namespace fmhf {
namespace {

constexpr int kRows = 128, kKeys = 128, kItemRows = 2 * kRows;
constexpr int kThreads = 11 * 32;   // 184 registers a thread: a softmax thread holds a row of S, 128 of them
constexpr uint32_t kTileChunk = 128 * 128;        // 128 rows of 64 columns
constexpr int kKernelPrompt = 6;                  // status codes 601..
constexpr int kLag = 8;
constexpr float kLazy = 8.f;                      // how far (in powers of two) the maximum may be exceeded before O is scaled again

template <int HD>
struct PromptCfg {
    static constexpr int kChunks = (HD + 63) / 64, kStages = HD == 64 ? 4 : 2;
    static constexpr bool kOverlay = HD != 64;    // P over S
    static constexpr uint32_t kTile = kChunks * kTileChunk;
    static constexpr uint32_t kOffQ = 0, kOffK = 2 * kTile, kOffV = kOffK + kStages * kTile, kOffBar = kOffV + kStages * kTile;
    static constexpr uint32_t kTotal = kOffBar + 512 + 1024;
    static constexpr uint32_t kColP = kOverlay ? 0 : 256, kPStride = kOverlay ? 128 : 64, kColO = kOverlay ? 256 : 384, kOStride = kOverlay ? 128 : 64;
};

// SFULL[g]: S computed; SFREE[g]: S in registers; PFULL[g]: P written, O scaled if need be; PVDONE[g]: the product that read P is done;
// OFULL[g]: the last of an item; OFREE[g]: O has been read out; ITEM*: the ring of work items.
enum { PB_QFULL = 0, PB_QEMPTY = 1, PB_SFULL = 2, PB_SFREE = 4, PB_PFULL = 6, PB_PVDONE = 8, PB_OFULL = 10, PB_OFREE = 12, PB_ITEMFULL = 14,
       PB_ITEMEMPTY = 16, PB_KFULL = 18, PB_KEMPTY = 22, PB_VFULL = 26, PB_VEMPTY = 30, PB_VRAW = 34, PB_COUNT = 38 };
static_assert(PB_COUNT * 8 + 16 + 2 * 48 + 32 <= 512, "control area");

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
    float scale, c;      // |scale| log2(e), at least a tiny number (masked scores are -inf, and 0 times that is not a number)
    int negate;          // scale < 0
    WaitArgs wait;
};

// Item `index`: the last rows of each sequence, which see the most keys when the call is causal, come first.  Sequence b owns the slots
// from cu[b] / 256 + b on, at least as many as it has tiles.
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

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
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

// A bounded wait of a whole warp, with the same answer for all lanes (those of a warp that gives up leave its loop together).  In line:
// a call would spill the row of S that a softmax thread holds.
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

// Turns at the special function unit of a quarter of the SM, which warps w and w + 4 share.  Left to themselves the two tiles fall into step:
// both take their exponentials at half speed and then wait for the tensor core together.  0: elsewhere, 1: wants it, 2: has it; of two
// that come together the first tile goes first.  A matter of speed only: whoever has waited 2000 clk goes ahead.
struct Turn {
    volatile int *mine, *other;
    int stop_at;                      // state of the other that this one waits for to end
    __device__ Turn(volatile int *turns, int warp) : mine(turns + warp), other(turns + (warp ^ 4)), stop_at(warp < 4 ? 2 : 1) {}
    __device__ __forceinline__ void take() {
        *mine = 1;
        const long long t0 = clock64();
        while (*other >= stop_at && clock64() - t0 < 2000) {}
        *mine = 2;
    }
    __device__ __forceinline__ void give() { *mine = 0; }
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const PromptArgs args) {
    using L = PromptCfg<HD>;
    constexpr int NS = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *gbase = smem_raw + (base - raw);
    const uint32_t sQ = base + L::kOffQ, sK = base + L::kOffK, sV = base + L::kOffV, sBar = base + L::kOffBar;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gbase + L::kOffBar + PB_COUNT * 8);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(gbase + L::kOffBar + PB_COUNT * 8 + 4);
    volatile int *items = reinterpret_cast<volatile int *>(gbase + L::kOffBar + PB_COUNT * 8 + 16);   // two of 12 words
    volatile int *turns = items + 24;                                                                 // eight: see Turn
    auto bar = [&](int i) { return sBar + 8u * i; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtl ctl{abort_flag, args.wait};
    constexpr int W = kKernelPrompt * 100;

    if (threadIdx.x == 0) {
        *abort_flag = launch_aborted(args.wait);
        mbar_init(bar(PB_QFULL), 1);
        mbar_init(bar(PB_QEMPTY), 2);
        for (int g = 0; g < 2; ++g) {
            mbar_init(bar(PB_SFULL + g), 1);
            mbar_init(bar(PB_SFREE + g), 4);
            mbar_init(bar(PB_PFULL + g), 4);
            mbar_init(bar(PB_PVDONE + g), 1);
            mbar_init(bar(PB_OFULL + g), 1);
            mbar_init(bar(PB_OFREE + g), 4);
            mbar_init(bar(PB_ITEMFULL + g), 1);
            mbar_init(bar(PB_ITEMEMPTY + g), 10);   // every warp but the one that fills it
        }
        for (int i = 0; i < 8; ++i) turns[i] = 0;
        for (int i = 0; i < NS; ++i) {
            mbar_init(bar(PB_KFULL + i), 1);
            mbar_init(bar(PB_KEMPTY + i), 2);
            mbar_init(bar(PB_VFULL + i), 1);
            mbar_init(bar(PB_VEMPTY + i), 2);
            mbar_init(bar(PB_VRAW + i), 1);
        }
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // The next work item, for a whole warp; false: give up.  `seq` counts the items of this CTA.
    auto next_item = [&](int seq, PromptItem &w) -> bool {
        const int s = seq & 1;
        if (!warp_wait(bar(PB_ITEMFULL + s), (seq >> 1) & 1, ctl, W + 1)) return false;
        volatile int *p = items + s * 12;
        w.q0 = p[0]; w.lq = p[1]; w.k0 = p[2]; w.lk = p[3]; w.see = p[4]; w.n0 = p[5]; w.n1 = p[6]; w.head = p[7];
        warp_arrive(bar(PB_ITEMEMPTY + s));
        return w.head >= 0;
    };

    if (*abort_flag) {
        // nothing: fall through to the teardown
    } else if (warp == 8) {
        // ------------------------------------------------------------------ work items and TMA
        if (lane == 0) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
            int seq = 0, n_q_loads = 0;
            uint32_t g = 0;          // tiles of keys so far
            bool ok = true;
            for (int index = blockIdx.x; ok; index += gridDim.x) {
                PromptItem w{};
                const bool last = index >= args.n_items;
                if (!last && !prompt_item(args, index, w)) continue;
                if (last) w.head = -1;
                const int s = seq & 1;
                if (seq >= 2 && !thread_wait(bar(PB_ITEMEMPTY + s), ((seq >> 1) - 1) & 1, ctl, W + 2)) break;
                volatile int *p = items + s * 12;
                p[0] = w.q0; p[1] = w.lq; p[2] = w.k0; p[3] = w.lk; p[4] = w.see; p[5] = w.n0; p[6] = w.n1; p[7] = w.head;
                mbar_arrive(bar(PB_ITEMFULL + s));
                ++seq;
                if (last) break;
                const int n = max(w.n0, w.n1);
                if (n == 0) continue;
                if (n_q_loads > 0 && !thread_wait(bar(PB_QEMPTY), (n_q_loads - 1) & 1, ctl, W + 3)) break;
                ++n_q_loads;
                mbar_arrive_expect_tx(bar(PB_QFULL), ((w.n0 > 0) + (w.n1 > 0)) * L::kTile);
                for (int t = 0; t < 2; ++t)
                    for (int c = 0; c < ((t ? w.n1 : w.n0) > 0 ? L::kChunks : 0); ++c)
                        tma_load_3d(sQ + t * L::kTile + c * kTileChunk, &tmQ, bar(PB_QFULL), c * 64, w.head, w.q0 + t * kRows);
                const int kh = w.head / args.group;
                for (int j = 0; j < n; ++j, ++g) {
                    const uint32_t st = g % NS, lap = (g / NS) & 1;
                    if (!thread_wait(bar(PB_KEMPTY + st), lap ^ 1, ctl, W + 4)) { ok = false; break; }
                    mbar_arrive_expect_tx(bar(PB_KFULL + st), L::kTile);
                    for (int c = 0; c < L::kChunks; ++c)
                        tma_load_3d(sK + st * L::kTile + c * kTileChunk, &tmK, bar(PB_KFULL + st), c * 64, kh, w.k0 + j * kKeys);
                    if (!thread_wait(bar(PB_VEMPTY + st), lap ^ 1, ctl, W + 5)) { ok = false; break; }
                    const uint32_t full = bar(((j + 1) * kKeys > w.lk ? PB_VRAW : PB_VFULL) + st);
                    mbar_arrive_expect_tx(full, L::kTile);
                    for (int c = 0; c < L::kChunks; ++c) tma_load_3d(sV + st * L::kTile + c * kTileChunk, &tmV, full, c * 64, kh, w.k0 + j * kKeys);
                }
            }
        }
    } else if (warp >= 9) {
        // ------------------------------------------------------------------ MMA issuers, one a tile of rows
        const int t = warp - 9;
        constexpr uint32_t idesc1 = umma_idesc(kRows, kKeys, false, false), idesc2 = umma_idesc(kRows, HD, false, true);
        const uint64_t dQ = desc_kmajor(sQ + t * L::kTile), dK0 = desc_kmajor(sK), dV0 = desc_mnmajor(sV, kTileChunk);
        const uint32_t tS = tmem + t * 128, tP = tmem + L::kColP + t * L::kPStride, tO = tmem + L::kColO + t * L::kOStride;
        PromptItem w;
        uint32_t g = 0, steps = 0;      // tiles of keys so far, of all items; those of this issuer's rows
        uint32_t ends = 0;              // parities of the stages' raw barriers, which only tiles with the end of a sequence use
        int loads = 0, outs = 0;
        bool ok = true;
        // S of tile j: its keys are there, S of the step before is in registers (and, over P, the product that read it done)
        auto scores = [&](int j, bool last) -> bool {
            const uint32_t st = (g + j) % NS, s = steps + j;
            if (!warp_wait(bar(PB_KFULL + st), ((g + j) / NS) & 1, ctl, W + 7)) return false;
            if (s > 0 && !warp_wait(bar((L::kOverlay ? PB_PVDONE : PB_SFREE) + t), (s - 1) & 1, ctl, W + 8)) return false;
            tc_fence_after();
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const uint32_t off = ((k >> 2) * kTileChunk + (k & 3) * 32) >> 4;
                    umma_ss(tS, dQ + off, dK0 + st * (L::kTile >> 4) + off, idesc1, k > 0 ? 1u : 0u);
                }
                umma_commit(bar(PB_KEMPTY + st));
                umma_commit(bar(PB_SFULL + t));
                if (last) umma_commit(bar(PB_QEMPTY));
            }
            __syncwarp();
            return true;
        };
        for (int seq = 0; ok && next_item(seq, w); ++seq) {
            const int n = max(w.n0, w.n1), mine = t ? w.n1 : w.n0;
            if (n == 0) continue;
            if (!warp_wait(bar(PB_QFULL), loads++ & 1, ctl, W + 9)) break;
            if (mine == 0 && lane == 0) mbar_arrive(bar(PB_QEMPTY));
            if (mine > 0 && !scores(0, mine == 1)) break;
            for (int j = 0; j < n; ++j) {
                const uint32_t st = (g + j) % NS, lap = ((g + j) / NS) & 1;
                if (t == 0 && (j + 1) * kKeys > w.lk) {
                    if (!warp_wait(bar(PB_VRAW + st), ends >> st & 1, ctl, W + 6)) { ok = false; break; }
                    ends ^= 1u << st;
                    for (int i = (w.lk - j * kKeys) * 8 + lane; i < kKeys * 8; i += 32)
#pragma unroll
                        for (int c = 0; c < L::kChunks; ++c) st_shared_v4(sV + st * L::kTile + c * kTileChunk + i * 16, 0, 0, 0, 0);
                    fence_async_smem();
                    warp_arrive(bar(PB_VFULL + st));
                }
                if (j >= mine) {       // the other tile of rows goes on alone: every phase is still seen, and every stage given back
                    if (!warp_wait(bar(PB_KFULL + st), lap, ctl, W + 10) || !warp_wait(bar(PB_VFULL + st), lap, ctl, W + 11)) { ok = false; break; }
                    if (lane == 0) {
                        mbar_arrive(bar(PB_KEMPTY + st));
                        mbar_arrive(bar(PB_VEMPTY + st));
                    }
                    continue;
                }
                if (!L::kOverlay && j + 1 < mine && !scores(j + 1, j + 2 == mine)) { ok = false; break; }
                if (!warp_wait(bar(PB_VFULL + st), lap, ctl, W + 12)) { ok = false; break; }
                if (j == 0 && outs > 0 && !warp_wait(bar(PB_OFREE + t), (outs - 1) & 1, ctl, W + 13)) { ok = false; break; }
                if (!warp_wait(bar(PB_PFULL + t), (steps + j) & 1, ctl, W + 14)) { ok = false; break; }
                tc_fence_after();
                if (lane == 0) {
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k) umma_ts(tO, tP + k * 8, dV0 + st * (L::kTile >> 4) + k * 128, idesc2, (j > 0 || k > 0) ? 1u : 0u);
                    umma_commit(bar(PB_VEMPTY + st));
                    umma_commit(bar(PB_PVDONE + t));
                    if (j + 1 == mine) umma_commit(bar(PB_OFULL + t));
                }
                __syncwarp();
                if (L::kOverlay && j + 1 < mine && !scores(j + 1, j + 2 == mine)) { ok = false; break; }
            }
            g += n;
            steps += mine;
            outs += mine > 0;
        }
    } else {
        // ------------------------------------------------------------------ softmax and output, a thread a row
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t tS = lanes + t * 128, tP = lanes + L::kColP + t * L::kPStride, tO = lanes + L::kColO + t * L::kOStride;
        const float c = args.c;
        Turn turn(turns, warp);
        PromptItem w;
        uint32_t steps = 0;
        int outs = 0;
        bool ok = true;
        for (int seq = 0; ok && next_item(seq, w); ++seq) {
            const int mine = t ? w.n1 : w.n0, r = t * kRows + row;
            const int see = args.causal ? max(0, min(w.lk, w.see + r)) : w.lk;      // keys that this row sees
            const int all = __shfl_sync(0xffffffffu, see, 0);                       // ... and every row of this warp
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < mine; ++j, ++steps) {
                if (!warp_wait(bar(PB_SFULL + t), steps & 1, ctl, W + 15)) { ok = false; break; }
                tc_fence_after();
                float s[128];
                tmem_ld32x2_sync(tS, tS + 32, reinterpret_cast<uint32_t *>(s), reinterpret_cast<uint32_t *>(s) + 32);
                tmem_ld32x2_sync(tS + 64, tS + 96, reinterpret_cast<uint32_t *>(s) + 64, reinterpret_cast<uint32_t *>(s) + 96);
                if (!L::kOverlay) {
                    tc_fence_before();
                    warp_arrive(bar(PB_SFREE + t));
                }
                if (args.negate)
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = -s[i];
                if ((j + 1) * kKeys > all) {
                    const int left = see - j * kKeys;
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i < left ? s[i] : -INFINITY;
                }
                float x = fmaxf(s[0], s[1]), y = fmaxf(s[2], s[3]);
#pragma unroll
                for (int i = 4; i < 128; i += 4) {
                    x = max3(x, s[i], s[i + 1]);
                    y = max3(y, s[i + 2], s[i + 3]);
                }
                x = fmaxf(x, y);
                // (the first finite maximum of a row is always taken: -inf is exceeded by more than anything)
                const bool raise = (x - m) * c > kLazy;
                if (__any_sync(0xffffffffu, raise)) {
                    const float now = fmaxf(m, x), keep = m == -INFINITY ? 0.f : ex2((m - now) * c);
                    m = now;
                    l *= keep;
                    if (j > 0) {
                        if (!L::kOverlay && !warp_wait(bar(PB_PVDONE + t), (steps - 1) & 1, ctl, W + 16)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll
                        for (int d = 0; d < HD; d += 16) {
                            uint32_t o[16];
                            tmem_ld16_sync(tO + d, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                            tmem_st16(tO + d, o);
                        }
                    }
                }
                const float mc = m == -INFINITY ? 0.f : -m * c;
                const f32x2 c2 = f2_pack(c, c), mc2 = f2_pack(mc, mc);
                f32x2 sum0 = 0, sum1 = 0;
                // the product of the step before has read P (over S it has: S could not have been computed else)
                if (!L::kOverlay && j > 0) {
                    if (!warp_wait(bar(PB_PVDONE + t), (steps - 1) & 1, ctl, W + 17)) { ok = false; break; }
                    tc_fence_after();
                }
                turn.take();
                // Exponents first, then exponentials with their sums and roundings eight behind: in program order nothing waits for the
                // result just asked for.
#pragma unroll
                for (int i = 0; i < 128; i += 2) f2_unpack(f2_fma(f2_pack(s[i], s[i + 1]), c2, mc2), s[i], s[i + 1]);
                uint32_t p[32];
#pragma unroll
                for (int i = 0; i < 128 + kLag; i += 4) {
                    if (i < 128) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) s[i + k] = ex2(s[i + k]);
                    }
                    if (i >= kLag) {
                        const int x = i - kLag;
                        sum0 = f2_add(sum0, f2_pack(s[x], s[x + 1]));
                        sum1 = f2_add(sum1, f2_pack(s[x + 2], s[x + 3]));
                        p[(x & 63) / 2] = pack_bf16(s[x], s[x + 1]);
                        p[(x & 63) / 2 + 1] = pack_bf16(s[x + 2], s[x + 3]);
                        if ((x & 63) == 60) tmem_st32(tP + (x >> 6) * 32, p);
                    }
                }
                turn.give();
                float a0, a1;
                f2_unpack(f2_add(sum0, sum1), a0, a1);
                l += a0 + a1;
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(bar(PB_PFULL + t));
            }
            if (!ok) break;
            if (mine > 0) {
                if (!warp_wait(bar(PB_OFULL + t), outs++ & 1, ctl, W + 18)) break;
                tc_fence_after();
            }
            const float inv = l > 0.f ? 1.f / l : 0.f;      // (NaN stays: l is not a number where a score is not)
            const bool mine_row = r < w.lq;
            __nv_bfloat16 *dst = args.o + (long long)(w.q0 + r) * args.o_tok + (long long)w.head * args.o_head;
#pragma unroll
            for (int d = 0; d < HD; d += 32) {
                uint32_t o[32];
                if (mine > 0) tmem_ld32_sync(tO + d, o);
                else
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                const float f = l != l ? l : inv;
                if (mine_row)
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            v[k] = l == 0.f ? 0u : pack_bf16(__uint_as_float(o[i + 2 * k]) * f, __uint_as_float(o[i + 2 * k + 1]) * f);
                        *reinterpret_cast<uint4 *>(dst + d + i) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
            }
            if (mine > 0) {
                tc_fence_before();
                warp_arrive(bar(PB_OFREE + t));
            }
            if (args.lse && mine_row)
                args.lse[(long long)(w.q0 + r) * args.n_q + w.head] = l == 0.f ? -INFINITY : (m * c + log2f(l)) * 0.6931471805599453f;
        }
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
    if (warp == 9) tmem_dealloc(tmem, 512);
}

template <int HD>
int launch_prompt(const flashmhf_prompt_attention_params &p, const PromptArgs &a, int num_sms, int device, cudaStream_t st, int *n_launch) {
    CUtensorMap q, k, v;
    auto map = [&](CUtensorMap *m, const void *ptr, const int64_t *stride, int heads, int tokens) {
        if (tokens == 0) heads = tokens = 1;      // no keys at all: nothing is read through the map
        const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)heads, (uint64_t)tokens};
        const int64_t str[2] = {stride[1], stride[0]};
        const uint32_t box[3] = {64, 1, 128};
        return encode_bf16_map(m, ptr, 3, dims, str, box);
    };
    int rc = map(&q, p.q, p.q_stride, p.n_q, p.tokens_q);
    if (rc == FLASHMHF_OK) rc = map(&k, p.k, p.k_stride, p.n_kv, p.tokens_k);
    if (rc == FLASHMHF_OK) rc = map(&v, p.v, p.v_stride, p.n_kv, p.tokens_k);
    if (rc != FLASHMHF_OK) return rc;
    const size_t smem = PromptCfg<HD>::kTotal;
    cudaError_t e = cudaSuccess;
    static std::atomic<bool> done[64];      // the attribute is per kernel and device
    if (!done[device].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(prompt_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        done[device].store(e == cudaSuccess, std::memory_order_release);
    }
    if (e == cudaSuccess)
        e = launch_kernel(false, prompt_attention_kernel<HD>, dim3((unsigned)(a.n_items < num_sms ? a.n_items : num_sms)), dim3(kThreads), smem, st, q, k, v, a);
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
    a.scale = p.scale;
    a.negate = p.scale < 0.f;
    const float c = (p.scale < 0.f ? -p.scale : p.scale) * 1.4426950408889634f;
    a.c = c > 1e-30f ? c : 1e-30f;
    a.wait = wait_args(&ctl);
    switch (p.head_dim) {
        case 64: return launch_prompt<64>(p, a, ctl.num_sms, ctl.device, st, n_launch);
        case 96: return launch_prompt<96>(p, a, ctl.num_sms, ctl.device, st, n_launch);
        default: return launch_prompt<128>(p, a, ctl.num_sms, ctl.device, st, n_launch);
    }
}

}  // namespace fmhf
