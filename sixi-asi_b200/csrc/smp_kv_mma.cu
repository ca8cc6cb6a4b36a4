// smp_kv_mma.cu - attention over the 8-bit paged cache on the tensor cores (sixi_kv_attend with bf16
// queries): the cached bytes go from memory to tcgen05.mma as they are, nothing is widened on the way.
//
// Mathematics. Both products are fp8 products with fp32 accumulation, and the 16-bit side of each is
// split into two e4m3 terms that are multiplied side by side:
//   S^T = K (q_hi + q_lo / 16)^T  a bf16 value has 8 significant bits, an e4m3 one has 4: after a row is
//                                 scaled by a power of two the split is exact (but for elements below
//                                 1/14,336 of the row's largest, which err by 2^-21.8 of it at most)
//   O^T = V^T (w_hi + w_lo / 32)  weights keep 8 significant bits, as bf16 weights would, down to 2^-13 of the largest of
//                                 their tile
// The scale of a page and head is a power of two, so it multiplies scores and weights exactly. Weights
// are scaled by a power of two per tile and row such that the tile's largest lies in (128, 256]; the tile's
// product is added to fp32 sums in registers with the factor taken out again, so a row whose running
// maximum lies far above a tile (a sink token) does not push that tile's weights below e4m3's range.
//
// A weight below 2^-13 of its tile's largest is off by 2^-21.6 of that at most (the last place of the low term, and of the
// weight's fp16 form), so the tile's 128 tokens together by 2^-14.6 of its sum. It shows only where the tokens with the
// large weights have values near zero and the others' sum is all that is left (fp32 queries keep it).
//
// Layout. Tokens are the M side of the scores (128 of them a tile, one per TMEM lane), query rows the N
// side (16 to 64: the query heads of one key head times new tokens); head elements are the M side of the
// output. So a decode step's 8 rows do not pad a 128-row tile, and K and V are both the A operand as they lie
// in memory: K is K-major, V MN-major, each a 128-byte-swizzled tile that TMA copies page by page (whatever
// the page size) into 128 x 128 bytes. The softmax reads scores in 16x256b fragments: a thread has 4 tokens of
// a quarter of the rows, so most of a row's maximum and sum is taken within a thread. The columns of the
// weights are dealt such that a thread's rows are neighbours there (row 8 j + 2 q + e is column
// q * R / 4 + 2 j + e), and go out in one store a token.
//
// A product of up to 128 columns takes about as long as one of 16 (40 to 66 cycles measured), so hi and lo are
// side by side in one operand of twice the rows, not two products.
//
// Roles, one CTA per SM: warps 0 and 3 copy the pages of keys and of values, warps 1 and 2 issue the two
// products, warps 4-7 keep the output's sums (one head element a thread), the next 8 or 12 are two or three
// softmax groups that take the tiles in turn, each with its own running maximum, and of the last 4 three stage
// queries (turned, split) and one walks the work and checks page tables. A tile's softmax is a chain of waits; two or three
// at a time, with the scores of the next ready before one ends, hide it.
//
// Bound and measured (one B200, bytes at its copy rate of 6.54 TB/s, products at 1.65 PFLOP/s):
//   64 sequences, one token, up to 16,000 cached, 32 heads on 8 of 128: 111 to 113 us, 5.4 to 5.5 TB/s (83 to 85 %
//     of the copy rate)
//   2 sequences, one token, up to 262,144 cached, 32 on 4 of 128:       92 to 95 us, 5.5 to 5.7 TB/s (84 to 87 %)
//   32 sequences, 9 tokens, up to 8,000 cached, 64 on 8 of 128:         178 to 194 us; 26 us of bytes
//   3 chunks of up to 2,048 tokens, window 4,096, 16 on 4 of 256:       772 to 794 us; 163 us of products
//   one token over 700 cached, 32 on 8 of 128:                          14 us, a chain of waits
// With few rows memory is the bound. With many rows a tile it is the softmax's chain of waits for scores, barriers and
// weights, and instruction fetch: 40 % of the issue slots, 28 % of the ALU and 17 % of the tensor pipe are busy, and code
// that is never run moves these times by 3 to 5 %.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "smp_kernels.cuh"
#include "smp_kv.cuh"

namespace sixi_b200 {
namespace {

constexpr int kTile = 128;      // tokens of a tile
constexpr int kTileShift = 7;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kWaitIters = 1u << 24;  // bound of a wait: a tenth of a second at the least (never expected to run out)
constexpr int kRing = 8;    // more than the tiles in flight, so that a waiter a few tiles behind finds its phase
constexpr uint32_t kPieces = 16; // piece records kept; the walk stays 12 ahead of the output at most
constexpr int kQSlots = 16;  // pieces whose row records are kept: softmax lags the staging by fewer than 10

// R columns for the rows of a row tile, of which the first 8 * NB are used, DC 128-element chunks of a head, G softmax
// groups
template <int R, int DC, int NB, int G>
struct Cfg {
    static constexpr int kThreads = 384 + 128 * G;
    // Registers of a thread by role: copies and products need few, output sums and softmax many. The shares of the
    // warpgroups add up to what the block is launched with (96 a thread for 5 warpgroups, 80 for 6).
    static constexpr int kRegsLaunch = G == 2 ? 96 : 80, kRegsIssue = 48, kRegsHelp = G == 2 ? 72 : 80;
    static constexpr int kRegsOut = G == 2 ? 136 : 88, kRegsSoft = G == 2 ? 112 : 88;
    static_assert(kRegsIssue + kRegsHelp + kRegsOut + G * kRegsSoft <= (3 + G) * kRegsLaunch, "registers");
    static constexpr int V = R / 4;                       // rows of a softmax thread
    static constexpr uint32_t kChunk = kTile * 128u;      // bytes of a tile's chunk of keys or values
    static constexpr uint32_t kBuf = DC * kChunk;
    static constexpr uint32_t kQ = DC * 2u * R * 128u;    // hi rows, lo rows, chunk by chunk
    static constexpr uint32_t kW = 2u * R * kTile;        // hi, lo
    static constexpr int kNQ = R == 16 ? 4 : 2;           // pieces whose queries are staged
    static constexpr uint32_t kFixed = kNQ * kQ + G * kW;
    static constexpr uint32_t kSmall = 7168u + (196u + 108u * G) * R;  // bound of the small arrays
    static constexpr int kBufs = static_cast<int>((227u * 1024u - 1024u - kSmall - kFixed) / kBuf);
    static constexpr int kNK = kBufs / 2 > 6 ? 6 : kBufs / 2;            // tiles of keys in flight
    static constexpr int kNV = kBufs - kNK > 6 ? 6 : kBufs - kNK;        // and of values
    static constexpr uint32_t kDyn = kFixed + (kNK + kNV) * kBuf + 1024u;
    static constexpr uint32_t kColsUsed = G * 2u * R * (1u + DC);  // scores and outputs, hi and lo, one of each a group
    static constexpr uint32_t kTmem = kColsUsed <= 64 ? 64u : (kColsUsed <= 128 ? 128u : (kColsUsed <= 256 ? 256u : 512u));
    static_assert(kNK >= 2 && kNV >= 2 && kColsUsed <= 512, "does not fit");
    static_assert(kRing > kNK && kRing > kNV, "a waiter's phase could come round again");
};

// ---------------------------------------------------------------------------------------------
// PTX

__device__ __forceinline__ uint32_t s32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(s32(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(s32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(s32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait of a whole warp. When a bound runs out anywhere in the CTA, no further wait waits and no further
// copy or product is issued: every role runs through its tiles and ends, and the results are reported as bad.
__device__ __forceinline__ void bar_wait(uint64_t* b, uint32_t parity, volatile uint32_t* gave_up) {
    if (!bar_try(b, parity)) {
        bool ok = false;
        for (uint32_t i = 0; i < kWaitIters && !ok; ++i) ok = bar_try(b, parity) || *gave_up != 0u;
        if (!ok) *gave_up = 1u;
    }
    __syncwarp();
}
// this warpgroup's registers a thread from `from` to `to`
template <int to, int from>
__device__ __forceinline__ void set_regs() {
    if constexpr (to > from) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(to));
    if constexpr (to < from) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(to));
}
// one lane of the (converged) warp: with it the compiler keeps the operands of a product uniform, which halves
// the cost of issuing one (40 cycles against 63 for a lane picked by its number)
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0u;
}
// Barrier of a softmax group's four warps. It is not bounded, but its warps cannot miss it: they run through the same
// tiles whatever happens to the waits, and agree on whatever they branch on around it (group_any): before each piece on
// whether there is one, in each tile on whether its scales differ.
__device__ __forceinline__ void group_sync(uint32_t grp) { asm volatile("bar.sync %0, 128;" ::"r"(2u + grp) : "memory"); }
__device__ __forceinline__ bool group_any(uint32_t grp, bool x) {
    uint32_t y;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(y)
        : "r"(x ? 1u : 0u), "r"(2u + grp)
        : "memory");
    return y != 0u;
}

__device__ __forceinline__ void tma_page(const CUtensorMap* map, void* dst, uint64_t* bar, int32_t x, int32_t z,
                                         uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, "
        "%5}], [%2], %6;" ::"r"(s32(dst)),
        "l"(map), "r"(s32(bar)), "r"(x), "r"(0), "r"(z), "l"(policy)
        : "memory");
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(b)) : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
// 8 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld8(uint32_t addr, float* x) {
    uint32_t v[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(addr));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[i]);
}
// a 16-lane, 8-column fragment: x[0..1] of lane (thread / 4), x[2..3] of lane 8 + (thread / 4), columns 2 * (thread % 4)..
__device__ __forceinline__ void tmem_ld_frag(uint32_t addr, float* x) {
    uint32_t v[4];
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(addr));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// shared-memory matrix descriptors: 128-byte swizzle (rows of 128 bytes, 8-row groups 1,024 bytes apart)
// and none (16-byte rows, 8-row groups `lead` bytes apart, 16-byte column groups `stride` bytes apart)
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_plain(uint32_t addr, uint32_t lead, uint32_t stride) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lead >> 4) << 16) |
           (static_cast<uint64_t>(stride >> 4) << 32) | (1ull << 46);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 operations at a time
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 un2(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// Two weights in [0, 1] as e4m3 codes of 256 times their value: hi = the nearest, lo = 32 times what hi leaves (8 at most).
// In f16, w has the exponent field that 256 w has in e4m3 (and subnormals have the same steps times 2^-7), so
// hi's code is w's f16 pattern rounded at bit 7. hi: the codes in bytes 0 and 2; lo: in bytes 0 and 1.
constexpr float kLoInv = 1.0f / 32.0f;
__device__ __forceinline__ void split2(F2 w, uint32_t* hi, uint32_t* lo) {
    const float2 f = un2(w);
    const __half2 h = __floats2half2_rn(f.x, f.y);
    const uint32_t top = (*reinterpret_cast<const uint32_t*>(&h) + 0x00400040u) & 0xFF80FF80u;
    const __half2_raw rest = __hmul2(__hsub2(h, *reinterpret_cast<const __half2*>(&top)), __float2half2_rn(8192.0f));
    *hi = top >> 7;
    *lo = __nv_cvt_halfraw2_to_fp8x2(rest, __NV_SATFINITE, __NV_E4M3);
}

// Over the 8 lanes of one lane % 4 (a thread's tokens): N values each, reduced to N / 8 (at least 1) a lane, value
// `first_of(lane)` on. Halves are exchanged and folded, so it takes N shuffles instead of 3 N.
template <int N, typename Op>
__device__ __forceinline__ void fold_lanes(float* x, uint32_t lane, Op op) {
    int n = N;
#pragma unroll
    for (int o = 16; o >= 4; o >>= 1) {
        const bool up = (lane & o) != 0u;
        if (n > 1) {
            n >>= 1;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                if (i >= n) break;
                const float send = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
                x[i] = op(keep, __shfl_xor_sync(0xFFFFFFFFu, send, o));
            }
        } else {
            x[0] = op(x[0], __shfl_xor_sync(0xFFFFFFFFu, x[0], o));
        }
    }
}
template <int N>
__device__ __forceinline__ uint32_t first_of(uint32_t lane) {
    if constexpr (N == 2) return lane >> 4;
    if constexpr (N == 4) return (lane >> 3) & 3u;
    if constexpr (N == 8) return lane >> 2;
    return (lane >> 2) * (N / 8);
}

// ---------------------------------------------------------------------------------------------

// A piece as the roles read it from shared memory: one warp walks this CTA's range and publishes them
struct PieceRec {
    uint64_t start;
    int64_t row0;
    uint32_t seq, head, row_tile, rows;  // rows = 0: no more pieces
    int32_t t0, t1, first, end;
    int32_t p0, len;
};
__device__ __forceinline__ PieceRec rec_of(bool any, const Piece& pc) {
    PieceRec r;
    r.start = pc.start, r.row0 = pc.plan.row0;
    r.seq = pc.seq, r.head = pc.head, r.row_tile = pc.row_tile, r.rows = any ? pc.rows : 0u;
    r.t0 = pc.t0, r.t1 = pc.t1, r.first = pc.first, r.end = pc.end;
    r.p0 = pc.plan.p0, r.len = pc.plan.len;
    return r;
}

template <int R, int DC, int NB, int G>
struct Shared {
    static constexpr int kNK = Cfg<R, DC, NB, G>::kNK, kNV = Cfg<R, DC, NB, G>::kNV, kNQ = Cfg<R, DC, NB, G>::kNQ;
    uint64_t kfull[kNK], vfull[kNV], scfull[kNV];
    uint64_t sfull[kRing], ofull[kRing];  // of tile n at n % kRing: its scores, its output are done
    uint64_t sempty[G], wfull[G], oempty[G], qfull[kNQ], qempty[kNQ], rfull[kQSlots], pfull[kPieces], lfull, lempty, done;
    unsigned long long scratch[Cfg<R, DC, NB, G>::kThreads / 32 + 2];
    SeqPlan found;
    PieceRec piece[kPieces], split[2];
    uint64_t total;
    uint32_t tmem, gave_up, ctas, pieces_done, split_mask, join_mask, disorder;
    float kscale[kNV][8], vscale[kNV][8];   // by page of the tile
    // by column of the weights:
    uint32_t frow[kQSlots][R];              // a row's factor from products to scores: score_factor's code
    int32_t qpos[kQSlots][R];               // a row's position
    float wmax[G][2][4][R];                 // [group][its tiles' parity][warp] a tile's maxima
    alignas(16) float2 ref[4 * G][R];       // [softmax warp] running maximum, weight factor; before: score factors
    float rescale[4 * G][R];                    // [softmax warp] factor of the older sums
    float osc[G][R], mgrp[G][R];            // a tile's factor, and the running maximum that its weights are under
    float2 sines[3][128];                   // [staging warp] of a token's pairs
    alignas(16) uint64_t row_at[4][R];      // [output warp] where a row goes
    alignas(16) float fac[4][R], facold[4][R];  // [output warp] a tile's factor, the older sums' factor
    float lsum[G][4][R], mfin[G][R];        // [group][warp] a piece's sums; [group] maxima
};

struct MmaArgs {
    AttnArgs a;
    uint32_t pages_per_tile;
    uint32_t read_once;  // no page is read by more than one row tile
    uint32_t out_pair;   // two elements of an output row can be stored together
    uint32_t q_vec;  // 8 query elements can be loaded (and are turned) together
};

// row of a column of the weights, and of the output
template <uint32_t V>
__device__ __forceinline__ constexpr uint32_t row_of(uint32_t col) {
    return ((col % V) >> 1) * 8u + (col / V) * 2u + (col & 1u);
}

// Queries are staged 8 elements a lane, DC * 16 lanes a row; a warp takes rows `at`, `at` + `step`, ... in units of the
// rows that it handles at once, U units at a time.
template <int DC>
__device__ __forceinline__ const __nv_bfloat16* query_row(const AttnArgs& a, const PieceRec& pc, uint32_t r, uint32_t* tok) {
    const uint32_t rr = pc.row_tile * a.shape.rt + r;
    *tok = rr / a.shape.group;
    return static_cast<const __nv_bfloat16*>(a.q.data) + (pc.row0 + *tok) * a.q.token_stride +
           (pc.head * a.shape.group + rr - *tok * a.shape.group) * a.q.head_stride;
}
template <int DC, int U>
__device__ __forceinline__ void fetch_queries(const MmaArgs& args, const PieceRec& pc, uint32_t rb, uint32_t step, uint4* raw) {
    constexpr uint32_t kRowLanes = DC * 16u, kAtOnce = 32u / kRowLanes;
    const uint32_t lane = threadIdx.x & 31u, d0 = (lane % kRowLanes) * 8u;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        uint32_t tok;
        const __nv_bfloat16* p =
            query_row<DC>(args.a, pc, min(rb + u * step * kAtOnce + lane / kRowLanes, pc.rows - 1u), &tok);
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (args.q_vec && d0 < args.a.g.head_dim) raw[u] = *reinterpret_cast<const uint4*>(p + d0);
    }
}

// A query's lo row holds 16 times what its hi row leaves: a query is up to 448 after scaling, so hi leaves 16 at most, and e4m3's
// last places reach 16 times further down.
constexpr float kLoQuery = 16.0f;

// A piece's queries as e4m3 hi and lo rows at dst (128-byte swizzle). raw: the first rows' elements, already asked for
// (fetch_queries); further ones are asked for a round ahead, as a load may take microseconds while the pages stream in.
// Sines cost most, and the rows of one token share them: where a warp's rows at a time belong to one token, its lanes
// work the token's pairs out between them, in tab (128 places of shared memory; NULL: none).
template <int R, int DC, int NB, int G, int U>
__device__ __forceinline__ void stage_queries(const MmaArgs& args, const PieceRec& pc, uint8_t* dst, uint32_t* frow, int32_t* qpos,
                                              uint32_t at, uint32_t step, float2* tab, uint4* raw) {
    constexpr uint32_t kRowLanes = DC * 16u, kAtOnce = 32u / kRowLanes, V = Cfg<R, DC, NB, G>::V;
    const AttnArgs& a = args.a;
    const uint32_t lane = threadIdx.x & 31u, D = a.g.head_dim;
    const uint32_t sub = lane / kRowLanes, d0 = (lane % kRowLanes) * 8u;
    const bool vec = args.q_vec != 0u, turn = a.rope.turns != nullptr, mine = d0 < D;
    const uint32_t half = a.rope.rot_dim >> 1, base = pc.row_tile * a.shape.rt, group = a.shape.group;
    uint32_t turned = 0xFFFFFFFFu;  // the token that tab holds
    for (uint32_t rb = at * kAtOnce; rb < pc.rows; rb += step * kAtOnce * U) {
        float x[U][8], m[U];
        const uint32_t tok0 = (base + rb) / group;
        const bool one = turn && tab != nullptr && vec &&
                         (base + min(rb + (U - 1u) * step * kAtOnce + kAtOnce - 1u, pc.rows - 1u)) / group == tok0;
        if (one && tok0 != turned) {
            __syncwarp();
            for (uint32_t i = lane; i < half; i += 32u) {
                float sn, cs;
                rope_sincos(a.rope, pc.p0 + static_cast<int32_t>(tok0), i, &sn, &cs);
                tab[i] = make_float2(cs, sn);
            }
            __syncwarp();
            turned = tok0;
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) unpack8(raw[u], x[u]);
        if (!vec || (turn && !one)) {
#pragma unroll 1
            for (uint32_t u = 0; u < U; ++u) {
                uint32_t tok;
                const __nv_bfloat16* p = query_row<DC>(a, pc, min(rb + u * step * kAtOnce + sub, pc.rows - 1u), &tok);
                float y[8];
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) y[j] = 0.0f;
                if (mine) {
#pragma unroll 1
                    for (uint32_t j = 0; j < 8; ++j) {
                        float z;
                        load_turned<__nv_bfloat16, 1>(a.rope, p, d0 + j, pc.p0 + static_cast<int32_t>(tok), &z);
#pragma unroll
                        for (uint32_t i = 0; i < 8; ++i)
                            if (i == j) y[i] = z;
                    }
                }
#pragma unroll
                for (uint32_t v = 0; v < U; ++v)
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j)
                        if (v == u) x[v][j] = y[j];
            }
        } else if (turn) {
            const bool upper = d0 >= half, turns = d0 < a.rope.rot_dim;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                float o[8];
                if (!a.rope.interleaved) {  // (the other halves are lanes of the same row)
                    const int from = static_cast<int>(lane) + (turns ? (upper ? -1 : 1) * static_cast<int>(half >> 3) : 0);
                    uint4 w;
                    w.x = __shfl_sync(0xFFFFFFFFu, raw[u].x, from), w.y = __shfl_sync(0xFFFFFFFFu, raw[u].y, from);
                    w.z = __shfl_sync(0xFFFFFFFFu, raw[u].z, from), w.w = __shfl_sync(0xFFFFFFFFu, raw[u].w, from);
                    unpack8(w, o);
                }
                if (!turns) continue;
                if (a.rope.interleaved) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float2 t = tab[(d0 + j) >> 1];
                        const float y = x[u][j] * t.x - x[u][j + 1] * t.y;
                        x[u][j + 1] = x[u][j + 1] * t.x + x[u][j] * t.y;
                        x[u][j] = y;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2 t = tab[(upper ? d0 - half : d0) + j];
                        x[u][j] = upper ? x[u][j] * t.x + o[j] * t.y : x[u][j] * t.x - o[j] * t.y;
                    }
                }
            }
        }
        if (rb + step * kAtOnce * U < pc.rows) fetch_queries<DC, U>(args, pc, rb + step * kAtOnce * U, step, raw);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            m[u] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // a turned query is rounded to its type, as a rotation of its own would be
                if (turn) x[u][j] = __bfloat162float(__float2bfloat16_rn(x[u][j]));
                const float ab = fabsf(x[u][j]);
                m[u] = ab < __builtin_huge_valf() ? fmaxf(m[u], ab) : __builtin_huge_valf();
            }
        }
#pragma unroll
        for (uint32_t o = kRowLanes / 2; o > 0; o >>= 1)
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) m[u] = fmaxf(m[u], __shfl_xor_sync(0xFFFFFFFFu, m[u], o));
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t r = rb + u * step * kAtOnce + sub;
            if (r >= pc.rows) continue;
            const bool bad = m[u] == __builtin_huge_valf();
            const int e = bad ? 0 : kv_scale_exp(m[u]);
            const float mul = exp2_int(-e) * a.score.sign;  // the sign of the scale is the query's here
            uint32_t h[2], l[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float v0 = x[u][4 * j] * mul, v1 = x[u][4 * j + 1] * mul;
                const float v2 = x[u][4 * j + 2] * mul, v3 = x[u][4 * j + 3] * mul;
                h[j] = e4m3x2(v0, v1) | (e4m3x2(v2, v3) << 16);
                const float2 h01 = e4m3x2_to_float2(h[j]), h23 = e4m3x2_to_float2(h[j] >> 16);
                l[j] = e4m3x2((v0 - h01.x) * kLoQuery, (v1 - h01.y) * kLoQuery) |
                       (e4m3x2((v2 - h23.x) * kLoQuery, (v3 - h23.y) * kLoQuery) << 16);
                if (bad) h[j] = 0x7F7F7F7Fu, l[j] = 0u;  // a NaN or Inf makes the row NaN
            }
            const uint32_t to = (d0 >> 7) * (2u * R * 128u) + r * 128u + ((((d0 & 127u) >> 4) ^ (r & 7u)) << 4) + (d0 & 8u);
            *reinterpret_cast<uint2*>(dst + to) = make_uint2(h[0], h[1]);
            *reinterpret_cast<uint2*>(dst + to + R * 128u) = make_uint2(l[0], l[1]);
            if (d0 == 0u) {
                const uint32_t col = ((r >> 1) & 3u) * V + (r >> 3) * 2u + (r & 1u);
                frow[col] = score_code(a.score, e);
                qpos[col] = pc.p0 + static_cast<int32_t>((base + r) / group);
            }
        }
    }
    fence_async_smem();
}

// Units that were cut: the last of their CTAs to arrive joins the pieces, in CTA order. The output's four warps and
// four of the softmax's do it (w: 0 to 7) after all of this CTA's own tiles, so that nothing of it waits for the
// joining.
template <int R, int DC, typename Sh>
__device__ __forceinline__ void join_pieces(const AttnArgs& a, Sh& sh, uint32_t w) {
    const uint32_t lane = threadIdx.x & 31u;
    __threadfence();
    asm volatile("bar.sync 14, 256;" ::: "memory");
    if (w == 0) {
        uint32_t joins = 0u;
        if (lane < 2u && (sh.split_mask & (1u << lane))) {
            const PieceRec& pc = sh.split[lane];
            const uint32_t c0 = place_owner(pc.start, sh.total, sh.ctas);
            const uint32_t c1 = place_owner(pc.start + static_cast<uint64_t>(pc.end - pc.first) - 1u, sh.total, sh.ctas);
            if (atomicAdd(a.counter + c0, 1u) == c1 - c0) {
                a.counter[c0] = 0u;
                joins = 1u << lane;
            }
        }
        joins = __reduce_or_sync(0xFFFFFFFFu, joins);
        if (lane == 0) sh.join_mask = joins;
    }
    asm volatile("bar.sync 14, 256;" ::: "memory");
    if (sh.join_mask == 0u) return;
    __threadfence();
    for (uint32_t mine = 0; mine < 2u; ++mine) {
        if (!(sh.join_mask & (1u << mine))) continue;
        const PieceRec& pc = sh.split[mine];
        const uint32_t c0 = place_owner(pc.start, sh.total, sh.ctas);
        const uint32_t n = place_owner(pc.start + static_cast<uint64_t>(pc.end - pc.first) - 1u, sh.total, sh.ctas) - c0 + 1u;
        const float* first = a.part + (2ull * c0 + 1u) * a.part_stride;       // the piece of c0 is its CTA's last
        const float* rest = a.part + (2ull * c0) * a.part_stride;             // the others' are their CTA's first
        join_rows<__nv_bfloat16, DC, R == 16 ? 2 : 4, R == 16 ? 4 / DC : 2 / DC>(a, first, rest, n, pc.rows, pc.row_tile * a.shape.rt, pc.row0, pc.head, w);
    }
}

template <int R, int DC, int NB, int G>
__global__ void __launch_bounds__(Cfg<R, DC, NB, G>::kThreads, 1)
    attend_mma_kernel(const __grid_constant__ MmaArgs args, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
    using C = Cfg<R, DC, NB, G>;
    constexpr int NK = C::kNK, NV = C::kNV, NQ = C::kNQ;
    constexpr uint32_t V = C::V, kStagers = C::kThreads / 32 - 2;
    // small row tiles are staged by one warp each, three at a time; large ones by three warps
    constexpr uint32_t kHelp = R == 16 ? 1 : 3;
    constexpr uint32_t kFull = 0xFFFFFFFFu;
    extern __shared__ uint8_t raw[];
    __shared__ Shared<R, DC, NB, G> sh;
    static_assert(sizeof(Shared<R, DC, NB, G>) <= C::kSmall, "small arrays");
    const AttnArgs& a = args.a;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t shift = a.g.page_shift, D = a.g.head_dim;
    uint8_t* dyn = raw + ((1024u - (s32(raw) & 1023u)) & 1023u);
    uint8_t* kbuf = dyn;
    uint8_t* vbuf = kbuf + NK * C::kBuf;
    uint8_t* qbuf = vbuf + NV * C::kBuf;
    uint8_t* wbuf = qbuf + NQ * C::kQ;
    volatile uint32_t* gave_up = &sh.gave_up;

    if (warp == 0) {
        if (lane < NK) bar_init(&sh.kfull[lane], 1);
        if (lane < NV) bar_init(&sh.vfull[lane], 1), bar_init(&sh.scfull[lane], 32);
        if (lane < kRing) bar_init(&sh.sfull[lane], 1), bar_init(&sh.ofull[lane], 1);
        if (lane < G) bar_init(&sh.sempty[lane], 4), bar_init(&sh.wfull[lane], 4), bar_init(&sh.oempty[lane], 4);
        if (lane < NQ) bar_init(&sh.qfull[lane], kHelp), bar_init(&sh.qempty[lane], 1);
        if (lane < kQSlots) bar_init(&sh.rfull[lane], kHelp);
        if (lane < kPieces) bar_init(&sh.pfull[lane], 1);
        if (lane == 0) {
            bar_init(&sh.lfull, 4 * G);
            bar_init(&sh.lempty, 4);
            bar_init(&sh.done, 2);
            sh.gave_up = sh.pieces_done = sh.split_mask = sh.disorder = 0u;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&sh.tmem)), "r"(C::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    PieceWalk walk;
    {
        uint64_t total;
        uint32_t ctas;
        tc_before();
        const bool busy = walk_init<C::kThreads>(a.shape, a.b, shift, sh.scratch, &sh.found, &sh.disorder, &walk, &total, &ctas);
        if (warp == C::kThreads / 32 - 1) {
            Piece pc;
            const bool any = busy && next_piece(a.shape, a.b, shift, walk, &pc);
            if (lane == 0) {
                sh.piece[0] = rec_of(any, pc);
                sh.total = total;
                sh.ctas = ctas;
                bar_arrive(&sh.pfull[0]);
            }
        }
        __syncthreads();
        tc_after();
    }
    const uint32_t tmem = sh.tmem;

    if (sh.piece[0].rows != 0u) {
        if (warp != 0 && warp != 3) {
            // the first piece's queries: by every warp but the copying ones, which start at once
            constexpr int kU = (8 * NB * DC / 2 + kStagers - 1) / kStagers;
            uint4 raw[kU];
            fetch_queries<DC, kU>(args, sh.piece[0], (warp - (warp > 3 ? 2u : 1u)) * (2u / DC), kStagers, raw);
            stage_queries<R, DC, NB, G, kU>(args, sh.piece[0], qbuf, sh.frow[0], sh.qpos[0], warp - (warp > 3 ? 2u : 1u), kStagers,
                                            nullptr, raw);
            asm volatile("bar.sync 15, %0;" ::"n"(C::kThreads - 64) : "memory");
        }
        // the next piece, or false after the last one
        const auto piece = [&](uint32_t np) -> const PieceRec* {
            bar_wait(&sh.pfull[np % kPieces], (np / kPieces) & 1u, gave_up);
            if (__any_sync(kFull, *gave_up != 0u) || sh.piece[np % kPieces].rows == 0u) return nullptr;
            return &sh.piece[np % kPieces];
        };
        if (warp < 4) {
            set_regs<C::kRegsIssue, C::kRegsLaunch>();
            if (warp == 0 || warp == 3) {
                // ---- pages: warp 0 copies the keys', warp 3 the values' and both's scales; a lane a page ----
                const bool is_v = warp == 3;
                const uint32_t ppt = args.pages_per_tile, n_buf = is_v ? NV : NK;
                const uint32_t none = a.g.n_pages * a.g.n_heads;  // a coordinate past the end: zeros
                const uint32_t slot = lane & 7u, window_mask = 32u / ppt - 1u;
                const CUtensorMap* map = is_v ? &v_map : &k_map;
                uint8_t* buf = is_v ? vbuf : kbuf;
                uint64_t* full = is_v ? sh.vfull : sh.kfull;
                uint64_t* done = is_v ? sh.ofull : sh.sfull;  // of tile n - n_buf: its buffer is free
                // pages that one row tile reads once leave L2 first: partial results and queries stay
                uint64_t policy;
                if (args.read_once) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
                else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
                uint32_t n = 0, st = 0;
                for (uint32_t np = 0; const PieceRec* rec = piece(np); ++np) {
                    const PieceRec& pc = *rec;
                    const int32_t* table = a.b.page_table + pc.seq * a.b.table_stride;
                    const uint32_t n_pg = (static_cast<uint32_t>(pc.len) + a.g.page_size - 1u) >> shift, head = pc.head;
                    uint32_t lo_pg = 0;  // pages wholly before the window of the unit's first row are not read
                    if (a.shape.window) {
                        const int32_t lo = pc.p0 + static_cast<int32_t>(pc.row_tile * a.shape.rt / a.shape.group) -
                                           static_cast<int32_t>(a.shape.window) + 1;
                        lo_pg = lo > 0 ? static_cast<uint32_t>(lo) >> shift : 0u;
                    }
                    // 32 page ids at a time, the next 32 asked for before they are needed
                    const uint32_t tiles = static_cast<uint32_t>(pc.t1 - pc.t0);
                    uint32_t idx = static_cast<uint32_t>(pc.t0) * ppt + lane;
                    int32_t ids = -1, ids_next = idx < n_pg && idx >= lo_pg ? table[idx] : -1;
                    for (uint32_t i = 0; i < tiles; ++i, ++n) {
                        const uint32_t in = i & window_mask;
                        if (in == 0) {
                            ids = ids_next;
                            idx += 32u;
                            ids_next = idx < n_pg && idx >= lo_pg ? table[idx] : -1;
                        }
                        const int32_t id = __shfl_sync(kFull, ids, in * ppt + (slot & (ppt - 1u)));
                        const bool good = static_cast<uint32_t>(id) < a.g.n_pages;
                        const uint32_t z = good ? static_cast<uint32_t>(id) * a.g.n_heads + head : none;
                        if (n >= n_buf) bar_wait(&done[(n - n_buf) % kRing], ((n - n_buf) / kRing) & 1u, gave_up);
                        if (__any_sync(kFull, *gave_up != 0u)) break;
                        if (lane == 0) bar_expect(&full[st], C::kBuf);
                        __syncwarp();
                        if (lane < ppt) {
#pragma unroll
                            for (int c = 0; c < DC; ++c)
                                tma_page(map, buf + st * C::kBuf + c * C::kChunk + slot * a.g.page_size * 128u, &full[st], c * 128, z, policy);
                        }
                        if (is_v) {
                            if (lane >= 16u) {
                                const float* src = (lane >= 24u ? a.g.v_scales : a.g.k_scales) + (good ? z : 0u);
                                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                                                 s32(lane >= 24u ? &sh.vscale[st][slot] : &sh.kscale[st][slot])),
                                             "l"(src), "r"(good ? 4u : 0u)
                                             : "memory");
                            }
                            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(s32(&sh.scfull[st])) : "memory");
                        }
                        if (++st == n_buf) st = 0;
                    }
                }
                if (*gave_up) {  // the copies in flight land before the shared memory is given back
                    for (uint32_t i = n > n_buf ? n - n_buf : 0u; i < n; ++i)
                        for (uint32_t w = 0; w < kWaitIters && !bar_try(&full[i % n_buf], (i / n_buf) & 1u); ++w) {}
                    asm volatile("cp.async.wait_all;" ::: "memory");
                }
            } else if (warp == 1) {
                // ---- scores: hi and lo rows of the queries are one operand of 2 R rows ----
                const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(R >> 2) << 17) | (8u << 24);
                const uint32_t ksteps = (D + 31u) / 32u;
                const uint64_t k_desc = desc_sw128(s32(kbuf)), q_desc = desc_sw128(s32(qbuf));
                uint32_t n = 0;
                for (uint32_t np = 0; const PieceRec* rec = piece(np); ++np) {
                    const PieceRec& pc = *rec;
                    const uint32_t qb = np % NQ;
                    bar_wait(&sh.qfull[qb], (np / NQ) & 1u, gave_up);
                    for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                        const uint32_t ks = n % NK, b = n % G;
                        bar_wait(&sh.kfull[ks], (n / NK) & 1u, gave_up);
                        if (n >= G) bar_wait(&sh.sempty[b], (n / G - 1u) & 1u, gave_up);
                        tc_after();
                        if (__any_sync(kFull, *gave_up != 0u)) continue;
                        const uint64_t kd = k_desc + ks * (C::kBuf >> 4), qd = q_desc + qb * (C::kQ >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < 4 * DC; ++k)
                                if (static_cast<uint32_t>(k) < ksteps)
                                    mma_f8(tmem + b * 2u * R, kd + (((k >> 2) * C::kChunk + (k & 3) * 32u) >> 4),
                                           qd + (((k >> 2) * (2u * R * 128u) + (k & 3) * 32u) >> 4), idesc, k > 0);
                        }
                        __syncwarp();
                        if (elect_one()) {
                            tc_commit(&sh.sfull[n % kRing]);
                            if (t + 1 == pc.t1) tc_commit(&sh.qempty[qb]);
                        }
                        __syncwarp();
                    }
                }
            } else {
                // ---- outputs: hi and lo columns of the weights are one operand of 2 R columns ----
                const uint32_t idesc = (1u << 4) | (1u << 15) | (1u << 16) | (static_cast<uint32_t>(R >> 2) << 17) | (8u << 24);
                const uint64_t v_desc = desc_sw128(s32(vbuf)), w_desc = desc_plain(s32(wbuf), 128u, 16u * kTile);
                uint32_t n = 0;
                for (uint32_t np = 0; const PieceRec* rec = piece(np); ++np) {
                    const PieceRec& pc = *rec;
                    for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                        const uint32_t vs = n % NV, b = n % G;
                        bar_wait(&sh.vfull[vs], (n / NV) & 1u, gave_up);
                        // (the softmax has waited for the output buffer to be free)
                        bar_wait(&sh.wfull[b], (n / G) & 1u, gave_up);
                        tc_after();
                        if (__any_sync(kFull, *gave_up != 0u)) continue;
                        const uint64_t vd = v_desc + vs * (C::kBuf >> 4), wd = w_desc + b * (C::kW >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int c = 0; c < DC; ++c)
#pragma unroll
                                for (int k = 0; k < kTile / 32; ++k)
                                    mma_f8(tmem + G * 2u * R + (b * DC + c) * 2u * R, vd + ((c * C::kChunk + k * 4096u) >> 4),
                                           wd + ((k * 512u) >> 4), idesc, k > 0);
                        }
                        __syncwarp();
                        if (elect_one()) tc_commit(&sh.ofull[n % kRing]);
                        __syncwarp();
                    }
                }
            }
        } else if (warp < 8) {
            set_regs<C::kRegsOut, C::kRegsLaunch>();
            // ---- output sums: thread d of a chunk holds element d of every row ----
            const uint32_t quad = warp & 3u, d0 = quad * 32u + lane;
            const uint32_t t_lane = tmem + ((quad * 32u) << 16) + G * 2u * R;
            constexpr int kPer = R > 32 ? 2 : 1;  // columns of a lane where columns are dealt to lanes
            float* fac = sh.fac[quad];
            float* facold = sh.facold[quad];
            uint32_t n = 0, np = 0;
            for (; const PieceRec* rec = piece(np); ++np) {
                const PieceRec& pc = *rec;
                F2 acc[DC][R / 2];
#pragma unroll
                for (int c = 0; c < DC; ++c)
#pragma unroll
                    for (int r = 0; r < R / 2; ++r) acc[c][r] = f2(0.0f, 0.0f);
                float M[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) M[i] = kNegInf;
                for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                    const uint32_t b = n % G;
                    // the weights' barrier orders the factors that the softmax wrote
                    bar_wait(&sh.wfull[b], (n / G) & 1u, gave_up);
                    bool changed = false;
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const uint32_t col = lane + 32u * i;
                        if (col < R && row_of<V>(col) < 8u * NB) {
                            const float mg = sh.mgrp[b][col], m1 = fmaxf(M[i], mg);
                            fac[col] = sh.osc[b][col] * (mg == m1 ? 1.0f : ex2(mg - m1));
                            const float al = M[i] == m1 ? 1.0f : ex2(M[i] - m1);
                            facold[col] = al;
                            changed |= al != 1.0f;
                            M[i] = m1;
                        }
                    }
                    changed = __any_sync(kFull, changed);
                    __syncwarp();
                    if (changed) {
#pragma unroll
                        for (int r = 0; r < R / 2; ++r) {
                            const float2 al = *reinterpret_cast<const float2*>(facold + 2 * r);
#pragma unroll
                            for (int c = 0; c < DC; ++c) acc[c][r] = mul2(acc[c][r], f2(al.x, al.y));
                        }
                    }
                    bar_wait(&sh.ofull[n % kRing], (n / kRing) & 1u, gave_up);
                    tc_after();
#pragma unroll
                    for (int r = 0; r < R; r += 8) {
                        if (row_of<V>(r) >= 8u * NB) continue;  // (the lowest row of the eight)
                        float o[DC][8], o_lo[DC][8];
#pragma unroll
                        for (int c = 0; c < DC; ++c) {
                            tmem_ld8(t_lane + (b * DC + c) * 2u * R + r, o[c]);
                            tmem_ld8(t_lane + (b * DC + c) * 2u * R + R + r, o_lo[c]);
                        }
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const float2 f = *reinterpret_cast<const float2*>(fac + r + j);
#pragma unroll
                            for (int c = 0; c < DC; ++c)
                                acc[c][(r + j) / 2] = fma2(fma2(f2(o_lo[c][j], o_lo[c][j + 1]), f2(kLoInv, kLoInv), f2(o[c][j], o[c][j + 1])),
                                                           f2(f.x, f.y), acc[c][(r + j) / 2]);
                        }
                    }
                    tc_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.oempty[b]);
                }
                bar_wait(&sh.lfull, np & 1u, gave_up);
                // the rows' sums, in facold; their maxima stay with the lanes, and go to fac
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const uint32_t col = lane + 32u * i;
                    if (col < R && row_of<V>(col) < 8u * NB) {
                        float l = 0.0f;
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const float mg = sh.mfin[g][col];
                            l += (sh.lsum[g][0][col] + sh.lsum[g][1][col] + sh.lsum[g][2][col] + sh.lsum[g][3][col]) *
                                 (mg == M[i] ? 1.0f : ex2(mg - M[i]));
                        }
                        facold[col] = l;
                        fac[col] = M[i];
                    }
                }
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.lempty);
                const bool whole = pc.t0 == pc.first && pc.t1 == pc.end;
                const uint32_t mine = (pc.t0 == pc.first ? 1u : 0u), rows = pc.rows;
                if (whole) {
                    // where each row goes: worked out by the lanes, a column each
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const uint32_t col = lane + 32u * i, r = row_of<V>(col);
                        if (col < R && r < pc.rows) {
                            const uint32_t tok = (pc.row_tile * a.shape.rt + r) / a.shape.group;
                            const uint32_t hq = pc.head * a.shape.group + (pc.row_tile * a.shape.rt + r) - tok * a.shape.group;
                            sh.row_at[quad][col] = (pc.row0 + tok) * a.out.token_stride + hq * a.out.head_stride;
                            if (a.lse && quad == 0)
                                a.lse[(pc.row0 + tok) * (a.shape.n_heads * a.shape.group) + hq] =
                                    (fac[col] + log2f(facold[col])) * kLn2;
                            facold[col] = facold[col] == 0.0f ? 0.0f : 1.0f / facold[col];  // (a row without positions: 0)
                        }
                    }
                    __syncwarp();
                    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out.data) + d0;
                    if (R == 16 && args.out_pair) {
                        // Two neighbours of a warp exchange halves of two rows: each stores two elements of one row. For small
                        // tiles only (64 sequences of one token: 113.6 us without, 111.2 with it): in the larger ones, which
                        // are bound by fetching instructions, the second form costs more than it saves (809 against 841 us
                        // for chunks of 32 rows of 256 elements).
                        const uint32_t odd = lane & 1u, sel = odd ? 0x3276u : 0x5410u;
                        out -= odd;
#pragma unroll
                        for (int col = 0; col < R; col += 2) {
                            if (row_of<V>(col) >= 8u * NB) continue;
                            const float2 inv = *reinterpret_cast<const float2*>(facold + col);
                            const uint64_t at = sh.row_at[quad][col + odd];
                            const bool on = row_of<V>(col) + odd < rows;
#pragma unroll
                            for (int c = 0; c < DC; ++c) {
                                const float2 y = un2(mul2(acc[c][col / 2], f2(inv.x, inv.y)));
                                const uint32_t two = bf16x2_bits(y.x, y.y);
                                const uint32_t w = __byte_perm(two, __shfl_xor_sync(kFull, two, 1), sel);
                                if (on && c * 128u + d0 < D) *reinterpret_cast<uint32_t*>(out + at + c * 128u) = w;
                            }
                        }
                    } else
                    // (four columns at a time: their places and factors are read together, the stores are predicated)
#pragma unroll
                    for (int col = 0; col < R; col += 4) {
                        if (row_of<V>(col) >= 8u * NB) continue;
                        const float4 inv = *reinterpret_cast<const float4*>(facold + col);
                        const float f[4] = {inv.x, inv.y, inv.z, inv.w};
                        const ulonglong2 at0 = *reinterpret_cast<const ulonglong2*>(&sh.row_at[quad][col]);
                        const ulonglong2 at1 = *reinterpret_cast<const ulonglong2*>(&sh.row_at[quad][col + 2]);
                        const uint64_t at[4] = {at0.x, at0.y, at1.x, at1.y};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int c = 0; c < DC; ++c) {
                                const float2 y = un2(acc[c][(col + i) / 2]);
                                const __nv_bfloat16 v = __float2bfloat16_rn(((i & 1) ? y.y : y.x) * f[i]);
                                if (row_of<V>(col + i) < rows && c * 128u + d0 < D) out[at[i] + c * 128u] = v;
                            }
                    }
                } else {
                    float* part = a.part + (2ull * blockIdx.x + mine) * a.part_stride + d0;
#pragma unroll
                    for (int col = 0; col < R; ++col) {
                        if (row_of<V>(col) >= 8u * NB) continue;
#pragma unroll
                        for (int c = 0; c < DC; ++c) {
                            const float2 y = un2(acc[c][col / 2]);
                            if (row_of<V>(col) < rows && c * 128u + d0 < D)
                                part[row_of<V>(col) * D + c * 128u] = (col & 1) ? y.y : y.x;
                        }
                    }
                    part -= d0;
                    if (quad == 0) {
#pragma unroll
                        for (int i = 0; i < kPer; ++i) {
                            const uint32_t col = lane + 32u * i, r = row_of<V>(col);
                            if (col < R && r < pc.rows) {
                                part[a.shape.rt * D + r] = fac[col];
                                part[a.shape.rt * (D + 1u) + r] = facold[col];
                            }
                        }
                    }
                    // at most two pieces of a CTA are parts of a unit: its first and its last
                    if (warp == 4 && lane == 0) {
                        sh.split[mine] = pc;
                        sh.split_mask |= 1u << mine;
                    }
                }
                __syncwarp();
                if (warp == 4 && lane == 0) *const_cast<volatile uint32_t*>(&sh.pieces_done) = np + 1u;
            }
            join_pieces<R, DC>(a, sh, warp - 4u);
        } else if (warp < 8 + 4 * G) {
            set_regs<C::kRegsSoft, C::kRegsLaunch>();
            // ---- softmax: group g takes the tiles n with n % G == g ----
            const uint32_t quad = warp & 3u, grp = (warp - 8u) >> 2, q = lane & 3u, tr = lane >> 2;
            const uint32_t t_lane = tmem + ((quad * 32u) << 16) + grp * 2u * R;
            const uint32_t pg0 = (quad * 32u) >> shift, pg1 = (quad * 32u + 16u) >> shift;
            constexpr int kFold = NB > 4 ? 16 : (NB > 2 ? 8 : 2 * NB);  // a thread's columns, to a power of two
            constexpr int kOwn = kFold > 8 ? kFold / 8 : 1;             // those that a lane ends with where they are dealt out
            const uint32_t own = q * V + first_of<kFold>(lane);
            float2* my_ref = sh.ref[warp - 8u];
            float* my_fac = reinterpret_cast<float*>(my_ref);  // (the same place, until the tile's maxima are known)
            float* my_rescale = sh.rescale[warp - 8u];
            uint8_t* w0 = wbuf + grp * C::kW + (quad * 4u) * 128u + tr * 16u + ((q * V) >> 4) * (16u * kTile) + ((q * V) & 15u);
            const auto max_op = [](float x, float y) { return fmaxf(x, y); };
            const auto add_op = [](float x, float y) { return x + y; };
            uint32_t n = 0;
            for (uint32_t np = 0;; ++np) {
                const PieceRec* rec = piece(np);
                if (group_any(grp, rec == nullptr)) break;
                const PieceRec& pc = *rec;
                const uint32_t rs = np % kQSlots;
                bar_wait(&sh.rfull[rs], (np / kQSlots) & 1u, gave_up);
                const int32_t* qpos = sh.qpos[rs] + q * V;
                // tiles in [safe_from, reach) are inside every row's positions
                const int32_t p_first = pc.p0 + static_cast<int32_t>(pc.row_tile * a.shape.rt / a.shape.group);
                const int32_t p_last = pc.p0 + static_cast<int32_t>((pc.row_tile * a.shape.rt + pc.rows - 1u) / a.shape.group);
                const int32_t reach = a.shape.all ? pc.len : min(pc.len, p_first + 1);
                const int32_t safe_from = a.shape.window ? p_last - static_cast<int32_t>(a.shape.window) + 1 : 0;
                float l[V];
#pragma unroll
                for (uint32_t i = 0; i < V; ++i) l[i] = 0.0f;
                float M[kOwn];
                uint32_t f_own[kOwn];
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    M[i] = kNegInf;
                    f_own[i] = sh.frow[rs][own + i];
                }
                for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                    if (n % G != grp) continue;
                    const uint32_t vs = n % NV, use = n / G;
                    float(*wmax)[R] = sh.wmax[grp][use & 1u];  // (its last readers met since)
                    bar_wait(&sh.scfull[vs], (n / NV) & 1u, gave_up);
                    const int ek0 = scale_exp_of(sh.kscale[vs][pg0]), ek1 = scale_exp_of(sh.kscale[vs][pg1]);
                    // From products to scores, base 2, by one factor a row and half of the warp's tokens (which may lie in
                    // two pages). A score is rounded here and nowhere later: the same value is compared and taken to its
                    // weight, so no weight is above 1 however large the scores are.
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) {
                        my_fac[own + i] = score_factor(f_own[i], ek0);
                        my_fac[R + own + i] = score_factor(f_own[i], ek1);
                    }
                    // exponents of the values' scales, relative to the tile's largest: they go into the weights.
                    // Where they differ by much, the weights' factor has to come from the largest product of
                    // weight and scale: the largest weight's own value could be below others' rounding.
                    const int ep = scale_exp_of(sh.vscale[vs][lane & (args.pages_per_tile - 1u)]);
                    int er = ep;
                    er = max(er, __shfl_xor_sync(kFull, er, 4));
                    er = max(er, __shfl_xor_sync(kFull, er, 2));
                    er = max(er, __shfl_xor_sync(kFull, er, 1));
                    const bool differ = __any_sync(kFull, ep > -127 && ep < er - 4);
                    const int ev0 = max(scale_exp_of(sh.vscale[vs][pg0]) - er, -126);
                    const int ev1 = max(scale_exp_of(sh.vscale[vs][pg1]) - er, -126);
                    const bool edge = t * kTile < safe_from || (t + 1) * kTile > reach;
                    bar_wait(&sh.sfull[n % kRing], (n / kRing) & 1u, gave_up);
                    tc_after();
                    float x[V / 2][2][4];  // [8-column block][column][token]
#pragma unroll
                    for (int j0 = 0; j0 < NB; j0 += 2) {  // (two blocks' loads under way)
                        float f[2][8], g[2][8];
#pragma unroll
                        for (int j = j0; j < j0 + 2; ++j) {
                            if (j >= NB) continue;
                            tmem_ld_frag(t_lane + 8 * j, f[j - j0]);
                            tmem_ld_frag(t_lane + (16u << 16) + 8 * j, f[j - j0] + 4);
                            tmem_ld_frag(t_lane + R + 8 * j, g[j - j0]);
                            tmem_ld_frag(t_lane + (16u << 16) + R + 8 * j, g[j - j0] + 4);
                        }
                        tmem_wait_ld();
#pragma unroll
                        for (int j = j0; j < j0 + 2; ++j) {
                            if (j >= NB) continue;
                            const float2 a0 = *reinterpret_cast<const float2*>(my_fac + q * V + 2 * j);
                            const float2 a1 = *reinterpret_cast<const float2*>(my_fac + R + q * V + 2 * j);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const F2 sum = fma2(f2(g[j - j0][2 * i], g[j - j0][2 * i + 1]), f2(1.0f / kLoQuery, 1.0f / kLoQuery),
                                                    f2(f[j - j0][2 * i], f[j - j0][2 * i + 1]));
                                const float2 y = un2(mul2(sum, i < 2 ? f2(a0.x, a0.y) : f2(a1.x, a1.y)));
                                x[j][0][i] = y.x, x[j][1][i] = y.y;
                            }
                        }
                    }
#pragma unroll
                    for (int j = NB; j < static_cast<int>(V / 2); ++j)  // columns without rows
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[j][0][i] = x[j][1][i] = kNegInf;
                    tc_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.sempty[grp]);
                    if (edge) {
                        const int32_t w = static_cast<int32_t>(a.shape.window);
#pragma unroll
                        for (int c = 0; c < static_cast<int>(V); ++c) {
                            const int32_t qp = qpos[c];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int32_t pos = t * kTile + static_cast<int32_t>(quad * 32u + i * 8u + tr);
                                bool ok = pos < pc.len && (a.shape.all || pos <= qp);
                                if (w) ok = ok && pos > qp - w;
                                if (!ok) x[c >> 1][c & 1][i] = kNegInf;
                            }
                        }
                    }
                    // the tile's maximum of every row: within the thread, over its warp, over the group
                    float mx[kFold];
#pragma unroll
                    for (int c = 0; c < kFold; ++c)
                        mx[c] = fmaxf(fmaxf(x[c >> 1][c & 1][0], x[c >> 1][c & 1][1]), fmaxf(x[c >> 1][c & 1][2], x[c >> 1][c & 1][3]));
                    fold_lanes<kFold>(mx, lane, max_op);
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) wmax[quad][own + i] = mx[i];
                    // (the group's warps agree on it: once waits have been given up, they may have read different scales, and
                    // a warp that went through the two barriers below alone would wait there for good)
                    const bool wide = group_any(grp, differ);
                    float mt[kOwn];
#pragma unroll
                    for (int i = 0; i < kOwn; ++i)
                        mt[i] = fmaxf(fmaxf(wmax[0][own + i], wmax[1][own + i]),
                                      fmaxf(wmax[2][own + i], wmax[3][own + i]));
                    float mw[kOwn];  // of weight times value scale
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) mw[i] = mt[i];
                    if (wide) {
#pragma unroll
                        for (int c = 0; c < kFold; ++c)
                            mx[c] = fmaxf(fmaxf(x[c >> 1][c & 1][0], x[c >> 1][c & 1][1]) + static_cast<float>(ev0),
                                          fmaxf(x[c >> 1][c & 1][2], x[c >> 1][c & 1][3]) + static_cast<float>(ev1));
                        fold_lanes<kFold>(mx, lane, max_op);
                        group_sync(grp);  // the first maxima have been read
#pragma unroll
                        for (int i = 0; i < kOwn; ++i) wmax[quad][own + i] = mx[i];
                        group_sync(grp);
#pragma unroll
                        for (int i = 0; i < kOwn; ++i)
                            mw[i] = fmaxf(fmaxf(wmax[0][own + i], wmax[1][own + i]),
                                          fmaxf(wmax[2][own + i], wmax[3][own + i]));
                    }
                    // weights e^(x - m1) times 2^k, k such that the tile's largest is in (1/2, 1]
                    bool changed = false;
                    float alpha[kOwn];
                    int k[kOwn];
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) {
                        const float m1 = fmaxf(M[i], mt[i]);
                        alpha[i] = M[i] == m1 ? 1.0f : ex2(M[i] - m1);
                        changed |= alpha[i] != 1.0f;
                        const float gap = m1 - mw[i];
                        k[i] = gap < 100.0f ? static_cast<int>(gap) : (mw[i] == kNegInf ? 0 : 100);
                        my_ref[own + i] = make_float2(m1 == kNegInf ? 0.0f : -m1, exp2_int(k[i]));
                        M[i] = m1;
                    }
                    changed = __any_sync(kFull, changed);
                    if (changed) {
#pragma unroll
                        for (int i = 0; i < kOwn; ++i) my_rescale[own + i] = alpha[i];
                        __syncwarp();
#pragma unroll
                        for (int c = 0; c < static_cast<int>(V); ++c) l[c] *= my_rescale[q * V + c];
                    }
                    __syncwarp();
                    if (use >= 1) bar_wait(&sh.ofull[(n - G) % kRing], ((n - G) / kRing) & 1u, gave_up);  // the weights' buffer is free
                    // all four tokens at a time, so that enough chains of exponential and rounding are under way; two for
                    // the largest row tile, whose bytes would not fit the registers
                    constexpr int kTok = NB > 5 ? 2 : 4, kWords = (NB + 1) / 2;
                    const float vr0 = exp2_int(ev0), vr1 = exp2_int(ev1);
#pragma unroll
                    for (int t0 = 0; t0 < 4; t0 += kTok) {
                        uint32_t hi[kTok][kWords], lo[kTok][kWords];
#pragma unroll
                        for (int j = 0; j < NB; ++j) {
                            const float4 rf = *reinterpret_cast<const float4*>(my_ref + q * V + 2 * j);
                            const F2 minus = f2(rf.x, rf.z);
                            const F2 wf0 = mul2(f2(rf.y, rf.w), f2(vr0, vr0)), wf1 = mul2(f2(rf.y, rf.w), f2(vr1, vr1));
                            F2 p[kTok];
#pragma unroll
                            for (int i = 0; i < kTok; ++i) {
                                const float2 y = un2(add2(f2(x[j][0][t0 + i], x[j][1][t0 + i]), minus));
                                p[i] = f2(ex2(y.x), ex2(y.y));
                            }
                            F2 sum = p[0];
#pragma unroll
                            for (int i = 1; i < kTok; ++i) sum = add2(sum, p[i]);
                            const float2 s2 = un2(add2(f2(l[2 * j], l[2 * j + 1]), sum));
                            l[2 * j] = s2.x, l[2 * j + 1] = s2.y;
#pragma unroll
                            for (int i = 0; i < kTok; ++i) {
                                uint32_t h, g;
                                split2(mul2(p[i], t0 + i < 2 ? wf0 : wf1), &h, &g);
                                if (j & 1) {
                                    hi[i][j / 2] = __byte_perm(hi[i][j / 2], h, 0x6420);
                                    lo[i][j / 2] = __byte_perm(lo[i][j / 2], g, 0x5410);
                                } else {  // (an odd block without a partner is packed here)
                                    hi[i][j / 2] = j + 1 < NB ? h : __byte_perm(h, 0u, 0x6420);
                                    lo[i][j / 2] = g;
                                }
                            }
                        }
                        const auto word = [&](const uint32_t(&w)[kWords], int k) { return k < kWords ? w[k < kWords ? k : 0] : 0u; };
#pragma unroll
                        for (int i = 0; i < kTok; ++i) {
                            uint8_t* wp = w0 + (t0 + i) * 128;
                            if constexpr (V == 4) {
                                *reinterpret_cast<uint32_t*>(wp) = hi[i][0];
                                *reinterpret_cast<uint32_t*>(wp + R * kTile) = lo[i][0];
                            } else if constexpr (V == 8) {
                                *reinterpret_cast<uint2*>(wp) = make_uint2(word(hi[i], 0), word(hi[i], 1));
                                *reinterpret_cast<uint2*>(wp + R * kTile) = make_uint2(word(lo[i], 0), word(lo[i], 1));
                            } else {
                                *reinterpret_cast<uint4*>(wp) =
                                    make_uint4(word(hi[i], 0), word(hi[i], 1), word(hi[i], 2), word(hi[i], 3));
                                *reinterpret_cast<uint4*>(wp + R * kTile) =
                                    make_uint4(word(lo[i], 0), word(lo[i], 1), word(lo[i], 2), word(lo[i], 3));
                            }
                        }
                    }
                    if (quad == 0) {
                        if (use >= 1) bar_wait(&sh.oempty[grp], (use - 1u) & 1u, gave_up);
#pragma unroll
                        for (int i = 0; i < kOwn; ++i) {
                            sh.osc[grp][own + i] = exp2_int(max(er, -126)) * exp2_int(-k[i] - 8);
                            sh.mgrp[grp][own + i] = M[i];
                        }
                    }
                    if ((t + 1) * kTile > pc.len) {
                        // what lies behind the sequence's end may hold NaN bytes, and 0 * NaN is NaN
                        bar_wait(&sh.vfull[vs], (n / NV) & 1u, gave_up);
                        const uint32_t tok = quad * 32u + lane;
                        if (t * kTile + static_cast<int32_t>(tok) >= pc.len) {
                            uint8_t* v = vbuf + vs * C::kBuf + tok * 128u;
#pragma unroll
                            for (int c = 0; c < DC; ++c)
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    *reinterpret_cast<uint4*>(v + c * C::kChunk + j * 16) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.wfull[grp]);
                }
                // the rows' sums over the warp's tokens
                fold_lanes<kFold>(l, lane, add_op);
                if (np >= 1) bar_wait(&sh.lempty, (np - 1u) & 1u, gave_up);
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    sh.lsum[grp][quad][own + i] = l[i];
                    if (quad == 0) sh.mfin[grp][own + i] = M[i];
                }
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.lfull);
            }
            if (grp == 0) join_pieces<R, DC>(a, sh, warp - 4u);
        } else {
            set_regs<C::kRegsHelp, C::kRegsLaunch>();
            if (warp == C::kThreads / 32 - 1) {
                // ---- the walk: pieces are published ahead of the roles ----
                for (uint32_t np = 1; sh.piece[(np - 1u) % kPieces].rows != 0u; ++np) {
                    Piece pc;
                    const bool any = next_piece(a.shape, a.b, shift, walk, &pc);
                    volatile uint32_t* done = &sh.pieces_done;
                    for (uint32_t i = 0; i < kWaitIters && np - *done > 12u && *gave_up == 0u; ++i)
                        __nanosleep(64);
                    __syncwarp();
                    if (__any_sync(kFull, np - *done > 12u)) break;  // (given up)
                    if (lane == 0) {
                        sh.piece[np % kPieces] = rec_of(any, pc);
                        bar_arrive(&sh.pfull[np % kPieces]);
                    }
                    // the piece's queries into L2: while the pages stream in, a load from memory takes some 5 us
                    if (any)
                        for (uint32_t i = lane; i < pc.rows * 4u; i += 32u) {
                            const uint32_t rr = pc.row_tile * a.shape.rt + (i >> 2), tok = rr / a.shape.group;
                            const uint32_t d = min((i & 3u) * 64u, D - 1u);
                            const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q.data) + (pc.plan.row0 + tok) * a.q.token_stride +
                                                     (pc.head * a.shape.group + rr - tok * a.shape.group) * a.q.head_stride + d;
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
                        }
                    __syncwarp();
                }
            } else {
                // ---- queries: of the pieces after the first ----
                const uint32_t h = warp - (8u + 4u * G);
                for (uint32_t np = 0; const PieceRec* rec = piece(np); ++np) {
                    if (kHelp == 1 && np % 3u != h) continue;
                    const uint32_t qb = np % NQ, rs = np % kQSlots;
                    constexpr int kU = R == 16 ? 4 : 3;
                    const uint32_t at = kHelp == 1 ? 0u : h;
                    uint4 raw[kU];
                    if (np > 0) fetch_queries<DC, kU>(args, *rec, at * (2u / DC), kHelp, raw);
                    if (np >= NQ) bar_wait(&sh.qempty[qb], (np / NQ - 1u) & 1u, gave_up);
                    if (np > 0)
                        stage_queries<R, DC, NB, G, kU>(args, *rec, qbuf + qb * C::kQ, sh.frow[rs], sh.qpos[rs], at, kHelp,
                                                        sh.sines[h], raw);
                    __syncwarp();
                    if (lane == 0) {
                        bar_arrive(&sh.qfull[qb]);
                        bar_arrive(&sh.rfull[rs]);
                    }
                }
            }
        }
    }
    if (warp == C::kThreads / 32 - 1) {
        // statuses, over the grid
        for (uint32_t s = blockIdx.x; s < a.b.n_seqs; s += gridDim.x) {
            const bool ok = sh.disorder == 0u && seq_pages_ok(a.shape, a.b, shift, a.g.n_pages, s, lane, 32u);
            const bool bad = __any_sync(kFull, !ok);
            if (lane == 0) {
                volatile int32_t* st = a.status + s;
                *st = bad ? SIXI_OUT_OF_BOUNDS : SIXI_OK;
                __threadfence();  // (a CTA that gives up raises the word first and writes its statuses after)
                if (*const_cast<volatile uint32_t*>(a.counter + kAttnMaxCtas)) *st = SIXI_BACKEND_ERROR;
            }
            __syncwarp();
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (sh.gave_up) {
        // never expected: the products in flight end (bounded) before their memory is given back
        if (warp == 1 || warp == 2) {
            if (elect_one()) {
                tc_commit(&sh.done);
                for (uint32_t w = 0; w < kWaitIters && !bar_try(&sh.done, 0u); ++w) {}
            }
            __syncwarp();
        }
        // the counters of the units that this CTA shares are not what they were: every later call reports it too
        if (tid == 0) *const_cast<volatile uint32_t*>(a.counter + kAttnMaxCtas) = 1u;
        __threadfence();
        __syncthreads();
        for (uint32_t s = tid; s < a.b.n_seqs; s += C::kThreads) *const_cast<volatile int32_t*>(a.status + s) = SIXI_BACKEND_ERROR;
    }
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
}

template <int R, int DC, int NB, int G>
cudaError_t launch(const MmaArgs& m, const CUtensorMap& k, const CUtensorMap& v, uint32_t rt, uint32_t n_sms,
                   cudaStream_t stream) {
    using C = Cfg<R, DC, NB, G>;
    static std::atomic<uint64_t> ready{0};  // the shared-memory opt-in is set once per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(attend_mma_kernel<R, DC, NB, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(C::kDyn));
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_acq_rel);
    }
    const uint32_t ctas = n_sms < kAttnMaxCtas ? n_sms : kAttnMaxCtas;
    MmaArgs args = m;
    args.a.shape.rt = rt;
    args.a.part_stride = part_floats(rt, m.a.g.head_dim);
    args.a.shape.tile_shift = kTileShift;
    args.a.shape.unit_cost = R == 16 ? 2u : 4u;
    // joining the pieces of a unit costs about as much as four tiles (one token over 700 cached ones, 32 heads on 8, 6 tiles
    // a unit: 13.9 us whole, 15.7 us cut)
    args.a.shape.whole_tiles = 8;
    attend_mma_kernel<R, DC, NB, G><<<ctas, C::kThreads, C::kDyn, stream>>>(args, k, v);
    return cudaGetLastError();
}

}  // namespace

cudaError_t make_page_map(void* pages, const KvGeom& g, CUtensorMap* out) {
    static std::atomic<void*> entry{nullptr};
    void* fn = entry.load(std::memory_order_acquire);
    if (fn == nullptr) {
        cudaDriverEntryPointQueryResult r;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &r);
        if (e != cudaSuccess) return e;
        if (r != cudaDriverEntryPointSuccess || fn == nullptr) return cudaErrorNotSupported;
        entry.store(fn, std::memory_order_release);
    }
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    // elements of a head, tokens of a page, page and head: one page of one head is a box (its rows padded
    // with zeros to 128 bytes, or two of them for heads beyond 128 elements)
    const cuuint64_t dims[3] = {g.head_dim, g.page_size, static_cast<cuuint64_t>(g.n_pages) * g.n_heads};
    const cuuint64_t strides[2] = {g.head_dim, static_cast<cuuint64_t>(g.head_dim) * g.page_size};
    const cuuint32_t box[3] = {128, g.page_size, 1};
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = reinterpret_cast<Encode>(fn)(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, pages, dims, strides, box, one,
                                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t launch_attend_bf16(const AttnArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map, uint32_t max_new,
                               uint32_t n_sms, cudaStream_t stream) {
    MmaArgs m;
    m.a = a;
    m.pages_per_tile = kTile / a.g.page_size;
    m.q_vec = ((reinterpret_cast<uintptr_t>(a.q.data) | 2u * a.q.token_stride | 2u * a.q.head_stride) & 15u) == 0 &&
                      rope_by_8(a.rope)
                  ? 1u
                  : 0u;
    m.out_pair = ((reinterpret_cast<uintptr_t>(a.out.data) | 2u * a.out.token_stride | 2u * a.out.head_stride) & 3u) == 0 ? 1u : 0u;
    const uint64_t rows = static_cast<uint64_t>(max_new ? max_new : 1u) * a.shape.group;
    // rows of a row tile: what deals `rows` out evenly, in the blocks of 8 rows that the softmax works in (72 rows
    // are 40 and 32, not 64 and 8)
    const uint64_t most = a.g.head_dim <= 128 ? 64 : 32, tiles = (rows + most - 1) / most;
    const uint32_t rt = static_cast<uint32_t>((((rows + tiles - 1) / tiles) + 7u) & ~7ull);
    m.read_once = rows <= rt ? 1u : 0u;
    // Beyond 32 rows the softmax is the bound and every 8 rows count, so each number of blocks has its own instance (32
    // sequences, up to 8,000 cached tokens, 8 key heads: 40 rows 103 us, 48 rows 112, 56 rows 138, 64 rows 150; by the
    // instance of 64 rows 143, 143, 154 and 150). Up to 32 rows memory is, and 24 rows do without (64.5 us by the
    // instance of 32 rows, 64.0 by one of their own).
    if (a.g.head_dim <= 128) {
        if (rt <= 8) return launch<16, 1, 1, 3>(m, k_map, v_map, rt, n_sms, stream);
        if (rt <= 16) return launch<16, 1, 2, 3>(m, k_map, v_map, rt, n_sms, stream);
        if (rt <= 32) return launch<32, 1, 4, 2>(m, k_map, v_map, rt, n_sms, stream);
        if (rt <= 40) return launch<64, 1, 5, 2>(m, k_map, v_map, rt, n_sms, stream);
        if (rt <= 48) return launch<64, 1, 6, 2>(m, k_map, v_map, rt, n_sms, stream);
        if (rt <= 56) return launch<64, 1, 7, 2>(m, k_map, v_map, rt, n_sms, stream);
        return launch<64, 1, 8, 2>(m, k_map, v_map, rt, n_sms, stream);
    }
    if (rt <= 8) return launch<16, 2, 1, 3>(m, k_map, v_map, rt, n_sms, stream);
    if (rt <= 16) return launch<16, 2, 2, 3>(m, k_map, v_map, rt, n_sms, stream);
    return launch<32, 2, 4, 2>(m, k_map, v_map, rt, n_sms, stream);
}

}  // namespace sixi_b200
