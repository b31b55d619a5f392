// Attention over packed prompts, bf16, sm_100a:  O = softmax(scale Q K^T + mask) V  per sequence and query head.
//
// A work item is a tile of 128 consecutive rows of one sequence and query head; it walks over its keys 128 at a time.  A step: the tensor
// core computes S = Q K^T (128 x 128, fp32 in tensor memory), a warpgroup (a thread a row) takes P = bf16(2^(c s - c r)), r a reference
// of the row near its maximum, into tensor memory, and the tensor core adds P V to O (fp32, in tensor memory over all steps): scores and
// weights never leave the SM.
//
// Bound: a chain of latencies, then the exponentials, then the way from L2.  The special function units take 1024 clk for the 128 x 128
// exponentials of a step and the two products 620 (a head of 64) to 1030 clk (128), but from S to P a step takes a warp some 3500 clk: tensor memory
// both ways, the maximum, barriers, and exponentials which a warp alone asks for at 68 % of the units' rate.  So two warpgroups take the
// steps in turn, with S and P in two buffers each.  Measured: 1770 (64) and 2000 clk (128) a step, special function units 53 % busy, tensor pipe 26
// and 50 %; 8192 causal tokens of 32 heads of 128 at 1.16 PFLOP/s (474 us) in a short loop, 0.97 to 1.0 (545 to 565 us) in a long one at the power limit.  What did not help: two tiles
// of rows a block (half the keys from L2, but tensor memory then has P only over S, and S waits for the product that reads P: 522 against 475 us with
// two warpgroups a tile), three warpgroups (the same reason: 547), four with 64 keys (a step costs each issuing thread 1000 clk whatever
// its size: 581), a cubic on the FMA pipe for a quarter of the exponentials (the same time), items in the order of their length and handed out one
// ahead (the order costs more than it gives: 56 -> 59 us for twelve ragged prompts, 139 -> 197 for 64 short ones).
//
// The reference is lazy: it is set to the maximum so far only where a row exceeds it by more than 2^16, and O is then multiplied by 2^(c r_old -
// c r_new).  P, its sum and O hold such values without loss (bf16 and fp32 are relative), so that almost no step touches O.  A step hands
// its reference on to the next one, in the other warpgroup, through shared memory.
//
// Work items are handed out by the hardware: the grid has a block for each (for some heads of each, where items are small), a resident block
// takes over one that has not started (clusterlaunchcontrol) while it works on its own.
//
// Warp roles: 0-3 and 4-7 softmax of the even and the odd steps (warp % 4 = TMEM lane quarter = 32 rows), 8 work items and TMA, 9 issues S, 10 O
// += P V and clears the rows of V behind the last key that a row of the item sees (a weight of 0 does not undo a NaN), 11 TMA of the values (heads above
// 64), 12-15 write out an item's rows while the others are at the next.
#include <atomic>

#include "paged.cuh"
#include "tc_common.cuh"
#include "tensormap.cuh"

namespace fmhf {
namespace {

constexpr int kRows = 128, kKeys = 128;
constexpr int kSoftmaxWarps = 8, kThreads = (kSoftmaxWarps + 8) * 32;
constexpr int kKernelPrompt = 6;                  // status codes 601..
constexpr float kLazy = 16.f;                     // how far (in powers of two) a row's reference may be exceeded before O is scaled to a new one
constexpr int kLag = 8;
constexpr int kMaxStages = 4;
constexpr uint32_t kControl = 768;
constexpr int kItems = 4;                             // work items that are known at a time

template <int HD>
struct PromptCfg {
    static constexpr int kChunks = (HD + 63) / 64, kStages = HD == 64 ? 4 : 2;
    static constexpr uint32_t kChunk = kRows * 128;             // 64 columns of a tile
    // With two stages the loader's thread waits for values while keys could go on: a warp of their own loads them (16 / 4 heads of 128:
    // 64 prompts of 300 rows 117 -> 99 us, 37 of 512 97 -> 89, 18 of 1024 121 -> 115, one of 8192 235 -> 236).  With four it seldom waits, and such a warp
    // only lets it take work further ahead than is well for the balance (heads of 64: 37 of 512 73 -> 76, 592 of 16 125 -> 140).
    static constexpr bool kValueWarp = kStages == 2;
    static_assert(kRows == kKeys, "tiles of Q, K and V are of one size");
    static constexpr uint32_t kTile = kChunks * kChunk;
    static constexpr uint32_t kOffQ = 0, kOffK = 2 * kTile, kOffV = kOffK + kStages * kTile;
    static constexpr uint32_t kOffMsg = kOffV + kStages * kTile, kOffEnd = kOffMsg + 2 * kRows * 4;   // [parity][row]: references; those and sums (of two items)
    static constexpr uint32_t kOffBar = kOffEnd + 2 * 2 * kRows * 8, kTotal = kOffBar + kControl + 1024;
};
// Tensor memory: two buffers for S, two for P (two bf16 a column), one for O, or two where there is room.
constexpr uint32_t kColP = 256, kColO = 384;
template <int HD>
constexpr int kOBufs = HD == 64 ? 2 : 1;

// SFULL: S computed into a buffer; SFREE: it is in registers; PFULL: P written, O scaled if need be; PVDONE: the product that read P is done (+
// buffer); OFULL: the last one of an item; OFREE: O has been read out (+ buffer); MSG: the reference that a step was taken with (quarter q, steps
// of parity b: + 2 q + b); ENDS, ENDSFREE: references and sums of an item's rows written, read; ITEM*: the ring of work items; NEXT: the answer
// to a request for one.
enum { PB_QFULL = 0, PB_QEMPTY = 2, PB_SFULL = 4, PB_SFREE = 6, PB_PFULL = 8, PB_PVDONE = 10, PB_OFULL = 12, PB_OFREE = 14, PB_ITEMFULL = 16,
       PB_ITEMEMPTY = PB_ITEMFULL + kItems, PB_ENDS = PB_ITEMEMPTY + kItems, PB_ENDSFREE = PB_ENDS + 2, PB_NEXT = PB_ENDSFREE + 2, PB_MSG = PB_NEXT + 1,
       PB_KFULL = PB_MSG + 8, PB_KEMPTY = PB_KFULL + kMaxStages,
       PB_VFULL = PB_KEMPTY + kMaxStages, PB_VEMPTY = PB_VFULL + kMaxStages, PB_VRAW = PB_VEMPTY + kMaxStages, PB_COUNT = PB_VRAW + kMaxStages };
constexpr uint32_t kOffNext = (PB_COUNT * 8 + 15) / 16 * 16, kOffItems = kOffNext + 16, kOffCtl = kOffItems + kItems * 48;
static_assert(kOffCtl + 8 <= kControl, "control area");

struct PromptItem {
    int q0, lq;          // first row of the item in the packed rows; rows of the sequence from there on
    int k0, lk;          // first key of the sequence, and keys from there on that the item's last row sees
    int see;             // keys that the item's first row sees, before clamping: row r sees min(lk, see + r) (causal) or lk
    int n;               // tiles of keys
    int head;            // -1: no more items
};

struct PromptArgs {
    __nv_bfloat16 *o;
    long long o_tok, o_head;
    float *lse;
    const int32_t *cu_q, *cu_k;
    int B, tokens_q, tokens_k, n_q, group, causal, heads, n_blocks;
    // scale log2(e) is c * before, c > 0: scores are multiplied by `before` as they come, and by c in the exponent, behind the mask.  `before` is the sign,
    // but where |scale| log2(e) is below 2^-60 it is all of it and c is 1: a c of 0 would make no number of a masked score's -inf.
    float c, before;
    int *index;
    WaitArgs wait;
};

// The first item of block `index` (which has a.heads of them, or what is left of n_q): the last rows of each sequence, which see the most keys when
// the call is causal, come first.  Sequence b owns the slots from cu[b] / 128 + b on, at least as many as it has items.
__device__ __forceinline__ bool prompt_item(const PromptArgs &a, int index, PromptItem &w) {
    const int slots = a.tokens_q / kRows + a.B, groups = (a.n_q + a.heads - 1) / a.heads, slot = slots - 1 - index / groups;
    w.head = index % groups * a.heads;
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(a.cu_q + mid) / kRows + mid <= slot) lo = mid;
        else hi = mid - 1;
    }
    const int q0 = __ldg(a.cu_q + lo), q1 = __ldg(a.cu_q + lo + 1), k0 = __ldg(a.cu_k + lo), k1 = __ldg(a.cu_k + lo + 1);
    if (q0 < 0 || q1 > a.tokens_q || q1 < q0 || k0 < 0 || k1 > a.tokens_k || k1 < k0) {
        note_index(a.index, kPromptRows);
        return false;
    }
    const int r0 = (slot - (q0 / kRows + lo)) * kRows, lq = q1 - q0, lk = k1 - k0;
    if (r0 < 0 || r0 >= lq) return false;
    w.q0 = q0 + r0;
    w.lq = lq - r0;
    w.k0 = k0;
    w.see = a.causal ? r0 + 1 + lk - lq : lk;
    // Keys behind those are nobody's here, like those behind the sequence: their values are cleared (a weight of 0 does not undo a NaN).  So a value
    // reaches rows of its own tile only, 127 before its own at most, wherever the tiles of keys begin.
    w.lk = a.causal ? min(lk, max(0, w.see + min(kRows, w.lq) - 1)) : lk;
    w.n = (w.lk + kKeys - 1) / kKeys;
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

// A thread's row of S, all of it behind one wait.
__device__ __forceinline__ void tmem_row(uint32_t ta, uint32_t *a) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%128];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%129];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(a[16]), "=r"(a[17]), "=r"(a[18]), "=r"(a[19]), "=r"(a[20]), "=r"(a[21]), "=r"(a[22]), "=r"(a[23]), "=r"(a[24]), "=r"(a[25]), "=r"(a[26]), "=r"(a[27]), "=r"(a[28]), "=r"(a[29]), "=r"(a[30]), "=r"(a[31]), "=r"(a[32]), "=r"(a[33]), "=r"(a[34]), "=r"(a[35]), "=r"(a[36]), "=r"(a[37]), "=r"(a[38]), "=r"(a[39]), "=r"(a[40]), "=r"(a[41]), "=r"(a[42]), "=r"(a[43]), "=r"(a[44]), "=r"(a[45]), "=r"(a[46]), "=r"(a[47]), "=r"(a[48]), "=r"(a[49]), "=r"(a[50]), "=r"(a[51]), "=r"(a[52]), "=r"(a[53]), "=r"(a[54]), "=r"(a[55]), "=r"(a[56]), "=r"(a[57]), "=r"(a[58]), "=r"(a[59]), "=r"(a[60]), "=r"(a[61]), "=r"(a[62]), "=r"(a[63]),
          "=r"(a[64]), "=r"(a[65]), "=r"(a[66]), "=r"(a[67]), "=r"(a[68]), "=r"(a[69]), "=r"(a[70]), "=r"(a[71]), "=r"(a[72]), "=r"(a[73]), "=r"(a[74]), "=r"(a[75]), "=r"(a[76]), "=r"(a[77]), "=r"(a[78]), "=r"(a[79]), "=r"(a[80]), "=r"(a[81]), "=r"(a[82]), "=r"(a[83]), "=r"(a[84]), "=r"(a[85]), "=r"(a[86]), "=r"(a[87]), "=r"(a[88]), "=r"(a[89]), "=r"(a[90]), "=r"(a[91]), "=r"(a[92]), "=r"(a[93]), "=r"(a[94]), "=r"(a[95]), "=r"(a[96]), "=r"(a[97]), "=r"(a[98]), "=r"(a[99]), "=r"(a[100]), "=r"(a[101]), "=r"(a[102]), "=r"(a[103]), "=r"(a[104]), "=r"(a[105]), "=r"(a[106]), "=r"(a[107]), "=r"(a[108]), "=r"(a[109]), "=r"(a[110]), "=r"(a[111]), "=r"(a[112]), "=r"(a[113]), "=r"(a[114]), "=r"(a[115]), "=r"(a[116]), "=r"(a[117]), "=r"(a[118]), "=r"(a[119]), "=r"(a[120]), "=r"(a[121]), "=r"(a[122]), "=r"(a[123]), "=r"(a[124]), "=r"(a[125]), "=r"(a[126]), "=r"(a[127])
        : "r"(ta), "r"(ta + 64)
        : "memory");
}

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
    volatile int *items = reinterpret_cast<volatile int *>(gbase + L::kOffBar + kOffItems);
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gbase + L::kOffBar + kOffCtl);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(gbase + L::kOffBar + kOffCtl + 4);
    auto bar = [&](int i) { return sBar + 8u * i; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtl ctl{abort_flag, args.wait};
    constexpr int W = kKernelPrompt * 100, kLoad = kSoftmaxWarps, kIssue = kLoad + 1, kValues = kLoad + 3, kOut = kLoad + 4;

    if (threadIdx.x == 0) {
        *abort_flag = launch_aborted(args.wait);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(PB_QFULL + i), 1);
            mbar_init(bar(PB_QEMPTY + i), 1);
            mbar_init(bar(PB_SFULL + i), 1);
            mbar_init(bar(PB_SFREE + i), 4);
            mbar_init(bar(PB_PFULL + i), 4);
            mbar_init(bar(PB_PVDONE + i), 1);
            mbar_init(bar(PB_OFULL + i), 1);
            mbar_init(bar(PB_OFREE + i), 4);
            mbar_init(bar(PB_ENDS + i), kSoftmaxWarps);
            mbar_init(bar(PB_ENDSFREE + i), 4);
        }
        for (int i = 0; i < kItems; ++i) {
            mbar_init(bar(PB_ITEMFULL + i), 1);
            mbar_init(bar(PB_ITEMEMPTY + i), kSoftmaxWarps + 6 + L::kValueWarp);      // softmax, both issuers, output
        }
        for (int i = 0; i < 8; ++i) mbar_init(bar(PB_MSG + i), 1);
        mbar_init(bar(PB_NEXT), 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(bar(PB_KFULL + i), 1);
            mbar_init(bar(PB_KEMPTY + i), 1);
            mbar_init(bar(PB_VFULL + i), 1);
            mbar_init(bar(PB_VEMPTY + i), 1);
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
    auto read_item = [&](unsigned seq, PromptItem &w) {
        volatile int *p = items + seq % kItems * 12;
        w.q0 = p[0]; w.lq = p[1]; w.k0 = p[2]; w.lk = p[3]; w.see = p[4]; w.n = p[5]; w.head = p[6];
    };
    auto next_item = [&](unsigned seq, PromptItem &w) -> bool {       // for a whole warp; false: no more, or given up
        if (!warp_wait(bar(PB_ITEMFULL + seq % kItems), seq / kItems & 1, ctl, W + 1)) return false;
        read_item(seq, w);
        warp_arrive(bar(PB_ITEMEMPTY + seq % kItems));
        return w.head >= 0;
    };

    // Tile j of an item's values, tile g of all; one thread.
    auto load_values = [&](uint32_t g, const PromptItem &w, int head, int j) -> bool {
        const uint32_t st = g % NS;
        if (!thread_wait(bar(PB_VEMPTY + st), (g / NS & 1) ^ 1, ctl, W + 5)) return false;
        const uint32_t full = bar(((j + 1) * kKeys > w.lk ? PB_VRAW : PB_VFULL) + st);
        mbar_arrive_expect_tx(full, L::kTile);
        for (int c = 0; c < L::kChunks; ++c) tma_load_3d(sV + st * L::kTile + c * L::kChunk, &tmV, full, c * 64, head, w.k0 + j * kKeys);
        return true;
    };

    if (*abort_flag) {
        // nothing: fall through to the teardown
    } else if (warp >= kOut) {
        // ------------------------------------------------------------------ output, a thread a row, while the other warps are at the next item
        // (registers: 256 x 208 for rows of S + 256 x 48 are the 512 x 128 that the launch has)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        const int row = (warp & 3) * 32 + lane;
        PromptItem w;
        int outs = 0;
        for (unsigned seq = 0; next_item(seq, w); ++seq) {
            if (!warp_wait(bar(PB_ENDS + (seq & 1)), (seq >> 1) & 1, ctl, W + 20)) break;
            // references and sums of both warpgroups: the larger reference is the later one
            volatile float2 *e = reinterpret_cast<volatile float2 *>(gbase + L::kOffEnd) + (seq & 1) * 2 * kRows + row;
            const float m0 = e[0].x, l0 = e[0].y, m1 = e[kRows].x, l1 = e[kRows].y, top = fmaxf(m0, m1), ref = top == -INFINITY ? 0.f : top;
            warp_arrive(bar(PB_ENDSFREE + (seq & 1)));
            const float l = l0 * ex2((m0 - ref) * args.c) + l1 * ex2((m1 - ref) * args.c);
            const bool none = top == -INFINITY && l < 1e-20f;      // (l is not a number, or not finite, where a score is not a number)
            const float inv = 1.f / l;
            const bool in = row < w.lq;
            const int ob = outs % kOBufs<HD>;
            const uint32_t tO = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kColO + ob * 64;
            if (w.n > 0) {
                if (!warp_wait(bar(PB_OFULL + ob), (outs / kOBufs<HD>) & 1, ctl, W + 19)) break;
                tc_fence_after();
                ++outs;
            }
            __nv_bfloat16 *dst = args.o + (long long)(w.q0 + row) * args.o_tok + (long long)w.head * args.o_head;
#pragma unroll
            for (int d = 0; d < HD; d += 16) {
                uint32_t o[16] = {};
                if (w.n > 0) tmem_ld16_sync(tO + d, o);
                if (in)
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        uint32_t v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            v[k] = none ? 0u : pack_bf16(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
                        *reinterpret_cast<uint4 *>(dst + d + i) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
            }
            if (w.n > 0) {
                tc_fence_before();
                warp_arrive(bar(PB_OFREE + ob));
            }
            if (args.lse && in) args.lse[(long long)(w.q0 + row) * args.n_q + w.head] = none ? -INFINITY : (top * args.c + log2f(l)) * 0.6931471805599453f;
        }
    } else if (warp >= kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == kLoad) {
            // -------------------------------------------------------------- work items and TMA
            if (lane == 0) {
                tma_prefetch_desc(&tmQ);
                tma_prefetch_desc(&tmK);
                tma_prefetch_desc(&tmV);
                unsigned seq = 0; int n_q = 0, asked = 0;
                uint32_t g = 0;          // tiles of keys so far
                bool ok = true;
                int index = blockIdx.x;
                const uint32_t answer = sBar + kOffNext;
                while (ok) {
                    // ask for the block after this one: the answer comes while this one is worked on
                    if (index >= 0) {
                        mbar_arrive_expect_tx(bar(PB_NEXT), 16);
                        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
                                     "r"(bar(PB_NEXT))
                                     : "memory");
                    }
                    PromptItem w{};
                    w.head = -1;
                    bool some = index < 0 || prompt_item(args, index, w);
                    const int last = index < 0 ? 0 : min(w.head + args.heads, args.n_q) - 1;
                    for (; ok && some; some = index >= 0 && w.head++ < last) {
                        const int s = seq % kItems;
                        if (seq >= kItems && !thread_wait(bar(PB_ITEMEMPTY + s), (seq / kItems - 1) & 1, ctl, W + 2)) { ok = false; break; }
                        volatile int *p = items + s * 12;
                        p[0] = w.q0; p[1] = w.lq; p[2] = w.k0; p[3] = w.lk; p[4] = w.see; p[5] = w.n; p[6] = w.head;
                        mbar_arrive(bar(PB_ITEMFULL + s));
                        ++seq;
                        if (index < 0) break;
                        const int n = w.head < 0 ? 0 : w.n;
                        if (n > 0) {
                            const int qb = n_q & 1;
                            if (n_q >= 2 && !thread_wait(bar(PB_QEMPTY + qb), ((n_q >> 1) - 1) & 1, ctl, W + 3)) { ok = false; break; }
                            ++n_q;
                            mbar_arrive_expect_tx(bar(PB_QFULL + qb), L::kTile);
                            for (int c = 0; c < L::kChunks; ++c)
                                tma_load_3d(sQ + qb * L::kTile + c * L::kChunk, &tmQ, bar(PB_QFULL + qb), c * 64, w.head, w.q0);
                        }
                        const int kh = w.head / args.group;
                        // keys of tile j, then (without a warp for them) values of tile j - 1, which are needed that much later: keys never wait for a
                        // stage of values
                        for (int j = 0; ok && j <= n && n > 0; ++j) {
                            if (j < n) {
                                const uint32_t st = (g + j) % NS;
                                if (!thread_wait(bar(PB_KEMPTY + st), ((g + j) / NS & 1) ^ 1, ctl, W + 4)) { ok = false; break; }
                                mbar_arrive_expect_tx(bar(PB_KFULL + st), L::kTile);
                                for (int c = 0; c < L::kChunks; ++c)
                                    tma_load_3d(sK + st * L::kTile + c * L::kChunk, &tmK, bar(PB_KFULL + st), c * 64, kh, w.k0 + j * kKeys);
                            }
                            if (!L::kValueWarp && j > 0) ok = load_values(g + j - 1, w, kh, j - 1);
                        }
                        g += n;
                    }
                    if (index < 0) break;
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
        } else if (L::kValueWarp && warp == kValues) {
            // -------------------------------------------------------------- TMA of the values
            if (lane == 0) {
                PromptItem w;
                uint32_t g = 0;           // tiles so far
                bool ok = true;
                for (unsigned seq = 0; ok; ++seq) {
                    if (!thread_wait(bar(PB_ITEMFULL + seq % kItems), seq / kItems & 1, ctl, W + 22)) break;
                    read_item(seq, w);
                    mbar_arrive(bar(PB_ITEMEMPTY + seq % kItems));
                    if (w.head < 0) break;
                    const int kh = w.head / args.group;
                    for (int j = 0; ok && j < w.n; ++j, ++g) ok = load_values(g, w, kh, j);
                }
            }
        } else if (warp == kIssue) {
            // -------------------------------------------------------------- S = Q K^T
            if (lane == 0) {
                constexpr uint32_t idesc = umma_idesc(kRows, kKeys, false, false);
                const uint64_t dQ0 = desc_kmajor(sQ), dK0 = desc_kmajor(sK);
                PromptItem w;
                uint32_t s = 0;           // steps so far, of all items
                int n_q = 0;
                bool ok = true;
                for (unsigned seq = 0; ok; ++seq) {
                    if (!thread_wait(bar(PB_ITEMFULL + seq % kItems), seq / kItems & 1, ctl, W + 8)) break;
                    read_item(seq, w);
                    mbar_arrive(bar(PB_ITEMEMPTY + seq % kItems));
                    if (w.head < 0) break;
                    if (w.n == 0) continue;
                    const int qb = n_q & 1;
                    if (!thread_wait(bar(PB_QFULL + qb), (n_q >> 1) & 1, ctl, W + 9)) break;
                    ++n_q;
                    for (int j = 0; j < w.n; ++j, ++s) {
                        const uint32_t st = s % NS, b = s & 1;
                        if (!thread_wait(bar(PB_KFULL + st), (s / NS) & 1, ctl, W + 10)) { ok = false; break; }
                        // its buffer is free: S of two steps before is in registers
                        if (s >= 2 && !thread_wait(bar(PB_SFREE + b), ((s >> 1) - 1) & 1, ctl, W + 11)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) {
                            const uint32_t off = (k >> 2) * L::kChunk + (k & 3) * 32;
                            umma_ss(tmem + b * kKeys, dQ0 + ((qb * L::kTile + off) >> 4), dK0 + ((st * L::kTile + off) >> 4), idesc, k > 0 ? 1u : 0u);
                        }
                        umma_commit(bar(PB_SFULL + b));
                        umma_commit(bar(PB_KEMPTY + st));
                        if (j + 1 == w.n) umma_commit(bar(PB_QEMPTY + qb));
                    }
                }
            }
        } else if (warp == kIssue + 1) {
            // -------------------------------------------------------------- O += P V
            constexpr uint32_t idesc = umma_idesc(kRows, HD, false, true);
            const uint64_t dV0 = desc_mnmajor(sV, L::kChunk);
            PromptItem w;
            uint32_t s = 0, seen = 0;      // steps so far; parities of the stages' raw barriers, which only tiles with the end of a sequence use
            int outs = 0;
            bool ok = true;
            for (unsigned seq = 0; ok && next_item(seq, w); ++seq) {
                const int ob = outs % kOBufs<HD>;
                for (int j = 0; j < w.n; ++j, ++s) {
                    const uint32_t st = s % NS, b = s & 1;
                    if ((j + 1) * kKeys > w.lk) {
                        if (!warp_wait(bar(PB_VRAW + st), seen >> st & 1, ctl, W + 7)) { ok = false; break; }
                        seen ^= 1u << st;
                        for (int i = (w.lk - j * kKeys) * 8 + lane; i < kKeys * 8; i += 32)
#pragma unroll
                            for (int c = 0; c < L::kChunks; ++c) st_shared_v4(sV + st * L::kTile + c * L::kChunk + i * 16, 0, 0, 0, 0);
                        fence_async_smem();
                        warp_arrive(bar(PB_VFULL + st));
                    }
                    if (!warp_wait(bar(PB_VFULL + st), (s / NS) & 1, ctl, W + 12)) { ok = false; break; }
                    if (j == 0 && outs >= kOBufs<HD> && !warp_wait(bar(PB_OFREE + ob), (outs / kOBufs<HD> - 1) & 1, ctl, W + 13)) { ok = false; break; }
                    if (!warp_wait(bar(PB_PFULL + b), (s >> 1) & 1, ctl, W + 14)) { ok = false; break; }
                    tc_fence_after();
                    if (lane == 0) {
#pragma unroll
                        for (int k = 0; k < kKeys / 16; ++k)
                            umma_ts(tmem + kColO + ob * 64, tmem + kColP + b * (kKeys / 2) + k * 8, dV0 + st * (L::kTile >> 4) + k * 128, idesc,
                                    (j > 0 || k > 0) ? 1u : 0u);
                        umma_commit(bar(PB_PVDONE + b));
                        umma_commit(bar(PB_VEMPTY + st));
                        if (j + 1 == w.n) umma_commit(bar(PB_OFULL + ob));
                    }
                    __syncwarp();
                }
                outs += w.n > 0;
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax, a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int par = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t tS = lanes + par * kKeys, tP = lanes + kColP + par * (kKeys / 2);
        const uint32_t msg_out = bar(PB_MSG + 2 * quarter + par), msg_in = bar(PB_MSG + 2 * quarter + (par ^ 1));
        volatile float *refs = reinterpret_cast<volatile float *>(gbase + L::kOffMsg) + row;
        volatile float2 *ends = reinterpret_cast<volatile float2 *>(gbase + L::kOffEnd) + par * kRows + row;
        const float c = args.c;
        PromptItem w;
        uint32_t steps = 0;
        int outs = 0;
        bool ok = true;
        for (unsigned seq = 0; ok && (ok = next_item(seq, w)); ++seq) {
            const int mine = w.n;
            const uint32_t tO = lanes + kColO + outs % kOBufs<HD> * 64;
            const int see = args.causal ? max(0, min(w.lk, w.see + row)) : w.lk;      // keys that this row sees
            const int all = __shfl_sync(0xffffffffu, see, 0);                       // ... and every row of this warp
            float m = -INFINITY, l = 0.f;      // the reference that this warpgroup's last step was taken with, and its weights' sum
            for (int j = (steps & 1) ^ par; j < mine; j += 2) {
                const uint32_t step = steps + j;
                if (!warp_wait(bar(PB_SFULL + par), (step >> 1) & 1, ctl, W + 18)) { ok = false; break; }
                tc_fence_after();
                float s[kKeys];
                tmem_row(tS, reinterpret_cast<uint32_t *>(s));
                tc_fence_before();
                warp_arrive(bar(PB_SFREE + par));
                // Asked here, needed behind the maximum: has the step before said what it was taken with?
                const bool heard = step == 0 || mbar_test(msg_in, ((step - 1) >> 1) & 1);
                if (args.before != 1.f)
#pragma unroll
                    for (int i = 0; i < kKeys; ++i) s[i] *= args.before;
                if ((j + 1) * kKeys > all) {
                    const int left = see - j * kKeys;
#pragma unroll
                    for (int i = 0; i < kKeys; ++i) s[i] = i < left ? s[i] : -INFINITY;
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < kKeys; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) top[k] = i + 4 < kKeys ? max3(top[k], s[i + k], s[i + 4 + k]) : fmaxf(top[k], s[i + k]);
                const float x = fmaxf(max3(top[0], top[1], top[2]), top[3]);
                if (!__all_sync(0xffffffffu, heard) && !warp_wait(msg_in, ((step - 1) >> 1) & 1, ctl, W + 16)) { ok = false; break; }
                const float was = j > 0 ? refs[(par ^ 1) * kRows] : -INFINITY;
                // (the first finite maximum of a row is always taken: -inf is exceeded by more than anything.  A row decides for itself: rows of
                // the next sequence, or of none, must not show in this one's last bits)
                const bool over = (x - was) * c > kLazy, any = __any_sync(0xffffffffu, over);
                const float ref = over ? x : was;
                refs[par * kRows] = ref;
                warp_arrive(msg_out);
                if (any && j > 0) {
                    // O is complete up to the step before.  One bit of parity tells a phase from the next one only: the product of two steps before
                    // is done, so P of three steps before has been written, so the next P of that parity is the one that is waited for; and who
                    // wrote that had waited for the product of three steps before.
                    if ((step > 1 && !warp_wait(bar(PB_PVDONE + par), ((step >> 1) - 1) & 1, ctl, W + 15)) ||
                        !warp_wait(bar(PB_PFULL + (par ^ 1)), ((step - 1) >> 1) & 1, ctl, W + 17) ||
                        !warp_wait(bar(PB_PVDONE + (par ^ 1)), ((step - 1) >> 1) & 1, ctl, W + 17)) { ok = false; break; }
                    tc_fence_after();
                    const float keep = was == ref ? 1.f : was == -INFINITY ? 0.f : ex2((was - ref) * c);
#pragma unroll
                    for (int d = 0; d < HD; d += 16) {
                        uint32_t o[16];
                        tmem_ld16_sync(tO + d, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                        tmem_st16(tO + d, o);
                    }
                }
                const float mc = ref == -INFINITY ? 0.f : -ref * c;
                const f32x2 c2 = f2_pack(c, c), mc2 = f2_pack(mc, mc);
                f32x2 sum0 = 0, sum1 = 0;
                uint32_t p[32];
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
                            p[((y + k) & 63) / 2] = pack_bf16(s[y + k], s[y + k + 1]);
                            p[((y + k) & 63) / 2 + 1] = pack_bf16(s[y + k + 2], s[y + k + 3]);
                        }
                        if (y == 56 && step > 1) {       // the product that read what P overwrites is done
                            ok = warp_wait(bar(PB_PVDONE + par), ((step >> 1) - 1) & 1, ctl, W + 15);
                            tc_fence_after();
                        }
                        if ((y & 63) == 56) tmem_st32(tP + y / 64 * 32, p);
                    }
                }
                if (!ok) break;
                float a0, a1;
                f2_unpack(f2_add(sum0, sum1), a0, a1);
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(bar(PB_PFULL + par));
                l = fmaf(l, m == ref ? 1.f : m == -INFINITY ? 0.f : ex2((m - ref) * c), a0 + a1);
                m = ref;
            }
            steps += mine;
            outs += mine > 0;
            if (!ok || (seq >= 2 && !(ok = warp_wait(bar(PB_ENDSFREE + (seq & 1)), ((seq >> 1) - 1) & 1, ctl, W + 21)))) break;
            volatile float2 *e = ends + (seq & 1) * 2 * kRows;
            e->x = m;
            e->y = l;
            warp_arrive(bar(PB_ENDS + (seq & 1)));
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
    if (warp == kIssue) tmem_dealloc(tmem, 512);
}

template <int HD>
int launch_prompt(const flashmhf_prompt_attention_params &p, const PromptArgs &a, int device, cudaStream_t st, int *n_launch) {
    CUtensorMap q, k, v;
    auto map = [&](CUtensorMap *m, const void *ptr, const int64_t *stride, int heads, int tokens) {
        if (tokens == 0) heads = tokens = 1;      // no keys at all: nothing is read through the map
        const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)heads, (uint64_t)tokens};
        const int64_t str[2] = {stride[1], stride[0]};
        const uint32_t box[3] = {64, 1, kRows};
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
    if (e == cudaSuccess) e = launch_kernel(false, prompt_attention_kernel<HD>, dim3((unsigned)a.n_blocks), dim3(kThreads), smem, st, q, k, v, a);
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
    // Heads of a block.  A block costs a request to the hardware and a search (2.7 us where there is one tile of keys in an item, 1.7 to 2.1 us an item with four
    // heads), but coarser ones share out long sequences worse.  us with 1 / 2 / 4 heads a block, 16 heads of 64: 592 prompts of 16 rows 188 / 136 / 125, 148 of 128
    // 65 / 52 / 50, 74 of 256 62 / 58 / 60, 37 of 512 73 / 75 / 82, twelve of 64 to 2048 86 / 101 / 131, 37 of 20 (four items an SM) 17 / 16 / 19.
    const long long slots = (long long)p.tokens_q / kRows + p.B, mean = p.tokens_q / p.B, items = slots * p.n_q;
    a.heads = mean <= 128 && items >= 16ll * ctl.num_sms ? 4 : mean <= 256 && items >= 8ll * ctl.num_sms ? 2 : 1;
    const long long blocks = slots * ((p.n_q + a.heads - 1) / a.heads);
    if (blocks > 0x3fffffffll) return FLASHMHF_ERR_BAD_SHAPE;
    a.n_blocks = (int)blocks;
    const float c = p.scale * 1.4426950408889634f, size = c < 0.f ? -c : c;
    const bool tiny = size < 0x1p-60f;
    a.c = tiny ? 1.f : size;
    a.before = tiny ? c : c < 0.f ? -1.f : 1.f;
    a.index = ctl.index;
    a.wait = wait_args(&ctl);
    switch (p.head_dim) {
        case 64: return launch_prompt<64>(p, a, ctl.device, st, n_launch);
        case 96: return launch_prompt<96>(p, a, ctl.device, st, n_launch);
        default: return launch_prompt<128>(p, a, ctl.device, st, n_launch);
    }
}

}  // namespace fmhf
