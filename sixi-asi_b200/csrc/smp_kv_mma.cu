// smp_kv_mma.cu - attention over the 8-bit paged cache on the tensor cores (sixi_kv_attend with bf16
// queries): the cached bytes go from memory to tcgen05.mma as they are, nothing is widened on the way.
//
// Mathematics. Both products are fp8 products with fp32 accumulation, and the 16-bit side of each is
// split into two e4m3 terms that are multiplied one after the other into the same accumulator:
//   S^T = K (q_hi + q_lo)^T       a bf16 value has 8 significant bits, an e4m3 one has 4: after a row is
//                                 scaled by a power of two the split is exact (but for elements below
//                                 1/1792 of the row's largest, which err by 2^-19 of it at most)
//   O^T = V^T (w_hi + w_lo)       weights keep 8 significant bits, as bf16 weights would
// The scale of a page and head is a power of two, so it multiplies scores and weights exactly. Weights
// are scaled by a power of two per tile and row such that the tile's largest lies in (128, 256]; the tile's
// product is added to fp32 sums in registers with the factor taken out again, so a row whose running
// maximum lies far above a tile (a sink token) does not push that tile's weights below e4m3's range.
//
// Weights below 2^-18 of the tile's largest lose bits, below 2^-23 they vanish: for a tile's 128 tokens
// together less than 2^-16 of its sum.
//
// Layout. Tokens are the M side of the scores (128 of them a tile, one per TMEM lane), query rows the N
// side (16 to 64: the query heads of one key head times new tokens); head elements are the M side of the
// output. So a decode step's 8 rows do not pad a 128-row tile, the softmax has one token per thread with
// all threads busy, and K and V are both the A operand as they lie in memory: K is K-major, V MN-major,
// each a 128-byte-swizzled tile that TMA copies page by page (whatever the page size) into 128 x 128 bytes.
//
// Roles, one CTA per SM: warp 0 copies pages, warp 1 issues the products, warps 2-3 stage queries (turned,
// split) and check page tables, warps 4-7 keep the output's sums (one head element a thread), warps 8-11
// (8-15 for 64 rows) are the softmax. Scores, weights and output tiles are double-buffered, so the
// products of one tile overlap the softmax of another; copies run up to 6 tiles ahead and across units.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "smp_kernels.cuh"
#include "smp_kv.cuh"

namespace sixi_b200 {
namespace {

constexpr int kTile = 128;      // tokens of a tile
constexpr int kTileShift = 7;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kWaitIters = 1u << 22;  // bound of every wait (never expected to run out)
constexpr int kQSlots = 8;  // pieces whose row records are kept: softmax lags the staging by fewer than 5

// R rows of a row tile, DC 128-element chunks of a head
template <int R, int DC>
struct Cfg {
    static constexpr int kGroups = R > 32 ? 2 : 1;        // softmax warpgroups
    static constexpr int kCols = R / kGroups;             // rows of one softmax warpgroup
    static constexpr int kThreads = 256 + 128 * kGroups;
    static constexpr uint32_t kChunk = kTile * 128u;      // bytes of a tile's chunk
    static constexpr uint32_t kStage = 2u * DC * kChunk;  // K then V
    static constexpr uint32_t kQ = DC * 2u * R * 128u;    // hi rows, lo rows, chunk by chunk
    static constexpr uint32_t kW = 2u * R * kTile;        // hi, lo
    static constexpr uint32_t kFixed = 2u * kQ + 2u * kW;
    static constexpr uint32_t kMax = 227u * 1024u - 1024u - 8192u;  // less alignment and the small arrays
    static constexpr int kFit = static_cast<int>((kMax - kFixed) / kStage);
    static constexpr int kStages = kFit > 6 ? 6 : kFit;
    static constexpr uint32_t kDyn = kFixed + kStages * kStage + 1024u;
    static constexpr uint32_t kColsUsed = 2u * R + 4u * DC * R;  // scores; hi and lo outputs; two of each
    static constexpr uint32_t kTmem = kColsUsed <= 64 ? 64u : (kColsUsed <= 128 ? 128u : (kColsUsed <= 256 ? 256u : 512u));
    static_assert(kStages >= 2 && kColsUsed <= 512, "does not fit");
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
// Bounded wait of a whole warp, with one answer for all its lanes: false when the bound ran out or
// another role of the CTA gave up.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile uint32_t* gave_up) {
    for (uint32_t i = 0; i < kWaitIters; ++i) {
        if (__all_sync(0xFFFFFFFFu, bar_try(b, parity))) return true;
        if (__any_sync(0xFFFFFFFFu, *gave_up != 0u)) return false;
    }
    *gave_up = 1u;
    return false;
}
// A bounded barrier of the warps that `b` counts (one arrival a warp); *phase is the caller's count.
__device__ __forceinline__ bool warps_meet(uint64_t* b, uint32_t* phase, volatile uint32_t* gave_up) {
    __syncwarp();
    if ((threadIdx.x & 31u) == 0) bar_arrive(b);
    const bool ok = bar_wait(b, *phase & 1u, gave_up);
    ++*phase;
    return ok;
}

__device__ __forceinline__ void tma_page(const CUtensorMap* map, void* dst, uint64_t* bar, int32_t x, int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            s32(dst)),
        "l"(map), "r"(s32(bar)), "r"(x), "r"(0), "r"(z)
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
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// Two weights in [0, 256] as e4m3 bytes: hi = the nearest, lo = what hi leaves, times 16. The rest is
// taken in f16 (11 significant bits; exact there, as hi is one of its values).
constexpr float kLoInv = 1.0f / 16.0f;
__device__ __forceinline__ void split2(float w0, float w1, uint32_t* hi, uint32_t* lo) {
    const __half2 w = __floats2half2_rn(w0, w1);
    const __half2_raw wr = w;
    const __nv_fp8x2_storage_t h = __nv_cvt_halfraw2_to_fp8x2(wr, __NV_SATFINITE, __NV_E4M3);
    const __half2 back = __half2(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3));
    const __half2_raw rest = __hmul2(__hsub2(w, back), __float2half2_rn(16.0f));
    *hi = h;
    *lo = __nv_cvt_halfraw2_to_fp8x2(rest, __NV_SATFINITE, __NV_E4M3);
}

// ---------------------------------------------------------------------------------------------

template <int R, int DC>
struct Shared {
    static constexpr int kS = Cfg<R, DC>::kStages;
    uint64_t kfull[kS], vfull[kS], empty[kS];
    uint64_t sfull[2], sempty[2], wfull[2], ofull[2], oempty[2], qfull[2], qempty[2], rfull[kQSlots], lfull, lempty, meet[3], done;
    unsigned long long scratch[Cfg<R, DC>::kThreads / 32 + 2];
    uint32_t tmem, gave_up, last_flag, pad;
    float kscale[kS][8], vscale[kS][8];     // by page of the tile
    float frow[kQSlots][R];                 // a row's factor from the product to the score, base 2
    int32_t qpos[kQSlots][R];               // a row's position; INT_MIN beyond the valid rows
    float wmax[2][R / Cfg<R, DC>::kCols][4][Cfg<R, DC>::kCols];
    float wmax2[Cfg<R, DC>::kGroups][4][Cfg<R, DC>::kCols];  // the same of weight times value scale
    float2 ref[Cfg<R, DC>::kGroups * 4][Cfg<R, DC>::kCols];  // per warp: running maximum, weight factor
    float osc[2][R], alpha[2][R];           // a tile's factor, and the older sums'
    uint32_t changed[2][2];                 // [buffer][group] some alpha is not 1
    float lsum[4][R], mfin[R];
};

struct MmaArgs {
    AttnArgs a;
    uint32_t pages_per_tile;
};

template <int R, int DC>
__global__ void __launch_bounds__(Cfg<R, DC>::kThreads, 1)
    attend_mma_kernel(const __grid_constant__ MmaArgs args, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
    using C = Cfg<R, DC>;
    constexpr int NS = C::kStages;
    extern __shared__ uint8_t raw[];
    __shared__ Shared<R, DC> sh;
    const AttnArgs& a = args.a;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t shift = a.g.page_shift, D = a.g.head_dim;
    uint8_t* dyn = raw + ((1024u - (s32(raw) & 1023u)) & 1023u);
    uint8_t* stages = dyn;
    uint8_t* qbuf = dyn + NS * C::kStage;
    uint8_t* wbuf = qbuf + 2u * C::kQ;
    volatile uint32_t* gave_up = &sh.gave_up;

    if (tid == 0) {
        for (int i = 0; i < NS; ++i) {
            bar_init(&sh.kfull[i], 33);  // the expected bytes, and the 32 lanes that copy scales
            bar_init(&sh.vfull[i], 1);
            bar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&sh.sfull[i], 1);
            bar_init(&sh.sempty[i], 4 * C::kGroups);
            bar_init(&sh.wfull[i], 4 * C::kGroups);
            bar_init(&sh.ofull[i], 1);
            bar_init(&sh.oempty[i], 4);
            bar_init(&sh.qfull[i], 2);
            bar_init(&sh.qempty[i], 1);
        }
        for (int i = 0; i < kQSlots; ++i) bar_init(&sh.rfull[i], 2);
        for (int i = 0; i < 3; ++i) bar_init(&sh.meet[i], 4);
        bar_init(&sh.lfull, 4 * C::kGroups);
        bar_init(&sh.lempty, 4);
        bar_init(&sh.done, 1);
        sh.gave_up = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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
    uint64_t total;
    uint32_t ctas;
    const bool busy = walk_init<C::kThreads>(a.shape, a.b, shift, sh.scratch, &walk, &total, &ctas);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = sh.tmem;

    if (busy) {
        Piece pc;
        if (warp == 0) {
            // ---- pages: one lane per page of a tile ----
            const uint32_t ppt = args.pages_per_tile;
            const uint32_t none = a.g.n_pages * a.g.n_heads;  // a coordinate past the end: zeros
            uint32_t n = 0;
            bool on = true;
            while (on && next_piece(a.shape, a.b, shift, walk, &pc)) {
                const int32_t* table = a.b.page_table + pc.seq * a.b.table_stride;
                const uint32_t n_pg = (static_cast<uint32_t>(pc.plan.len) + a.g.page_size - 1u) >> shift;
                uint32_t lo_pg = 0;  // pages wholly before the window of the unit's first row are not read
                if (a.shape.window) {
                    const int32_t lo = pc.plan.p0 + static_cast<int32_t>(pc.row_tile * R / a.shape.group) -
                                       static_cast<int32_t>(a.shape.window) + 1;
                    lo_pg = lo > 0 ? static_cast<uint32_t>(lo) >> shift : 0u;
                }
                // page ids a tile ahead
                const uint32_t slot = lane & 7u;
                uint32_t idx = static_cast<uint32_t>(pc.t0) * ppt + slot;
                int32_t id = slot < ppt && idx < n_pg && idx >= lo_pg ? table[idx] : -1;
                for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                    const uint32_t st = n % NS;
                    const bool good = static_cast<uint32_t>(id) < a.g.n_pages;
                    const uint32_t z = good ? static_cast<uint32_t>(id) * a.g.n_heads + pc.head : none;
                    idx += ppt;
                    id = t + 1 < pc.t1 && slot < ppt && idx < n_pg && idx >= lo_pg ? table[idx] : -1;
                    if (n >= NS && !bar_wait(&sh.empty[st], ((n / NS) - 1u) & 1u, gave_up)) {
                        on = false;
                        break;
                    }
                    uint8_t* dst = stages + st * C::kStage;
                    if (lane == 0) {
                        bar_expect(&sh.kfull[st], DC * C::kChunk);
                        bar_expect(&sh.vfull[st], DC * C::kChunk);
                    }
                    __syncwarp();
                    if (lane < 8u) {
                        if (slot < ppt) {
#pragma unroll
                            for (int c = 0; c < DC; ++c)
                                tma_page(&k_map, dst + c * C::kChunk + slot * a.g.page_size * 128u, &sh.kfull[st], c * 128, z);
                        }
                    } else if (lane < 16u) {
                        if (slot < ppt) {
#pragma unroll
                            for (int c = 0; c < DC; ++c)
                                tma_page(&v_map, dst + (DC + c) * C::kChunk + slot * a.g.page_size * 128u, &sh.vfull[st],
                                         c * 128, z);
                        }
                    } else {
                        const bool is_v = lane >= 24u;
                        const float* src = (is_v ? a.g.v_scales : a.g.k_scales) + (good ? z : 0u);
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                                         s32(is_v ? &sh.vscale[st][slot] : &sh.kscale[st][slot])),
                                     "l"(src), "r"(good ? 4u : 0u)
                                     : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(s32(&sh.kfull[st])) : "memory");
                }
            }
            if (*gave_up) {  // the copies in flight land before the shared memory is given back
                for (uint32_t i = n > NS ? n - NS : 0u; i < n; ++i) {
                    for (uint32_t w = 0; w < kWaitIters && !bar_try(&sh.kfull[i % NS], (i / NS) & 1u); ++w) {}
                    for (uint32_t w = 0; w < kWaitIters && !bar_try(&sh.vfull[i % NS], (i / NS) & 1u); ++w) {}
                }
            }
        } else if (warp == 1) {
            // ---- products: the scores of tile n, then the output of tile n - 1 ----
            const uint32_t idesc_s = (1u << 4) | (static_cast<uint32_t>(R >> 3) << 17) | (8u << 24);
            const uint32_t idesc_o = (1u << 4) | (1u << 15) | (1u << 16) | (static_cast<uint32_t>(R >> 2) << 17) | (8u << 24);
            const uint32_t ksteps = (D + 31u) / 32u;
            uint32_t n = 0, np = 0;
            bool on = true;
            auto output = [&](uint32_t m) {
                const uint32_t st = m % NS, b = m & 1u;
                if (!bar_wait(&sh.vfull[st], (m / NS) & 1u, gave_up)) return false;
                if (!bar_wait(&sh.wfull[b], (m >> 1) & 1u, gave_up)) return false;
                if (m >= 2 && !bar_wait(&sh.oempty[b], ((m >> 1) - 1u) & 1u, gave_up)) return false;
                tc_after();
                if (lane == 0) {
                    const uint32_t v = s32(stages + st * C::kStage + DC * C::kChunk), w = s32(wbuf + b * C::kW);
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const uint32_t d = tmem + 2u * R + (b * DC + c) * 2u * R;
#pragma unroll
                        for (int k = 0; k < kTile / 32; ++k)
                            mma_f8(d, desc_sw128(v + c * C::kChunk + k * 4096u), desc_plain(w + k * 512u, 128u, 16u * kTile),
                                   idesc_o, k > 0);
                    }
                    tc_commit(&sh.ofull[b]);
                    tc_commit(&sh.empty[st]);
                }
                __syncwarp();
                return true;
            };
            while (on && next_piece(a.shape, a.b, shift, walk, &pc)) {
                const uint32_t qb = np & 1u;
                if (!bar_wait(&sh.qfull[qb], (np >> 1) & 1u, gave_up)) break;
                for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                    const uint32_t st = n % NS, b = n & 1u;
                    on = bar_wait(&sh.kfull[st], (n / NS) & 1u, gave_up) &&
                         (n < 2 || bar_wait(&sh.sempty[b], ((n >> 1) - 1u) & 1u, gave_up));
                    if (!on) break;
                    tc_after();
                    if (lane == 0) {
                        const uint32_t k0 = s32(stages + st * C::kStage), q0 = s32(qbuf + qb * C::kQ);
                        for (uint32_t part = 0; part < 2; ++part)
                            for (uint32_t k = 0; k < ksteps; ++k)
                                mma_f8(tmem + b * R, desc_sw128(k0 + (k >> 2) * C::kChunk + (k & 3u) * 32u),
                                       desc_sw128(q0 + (k >> 2) * (2u * R * 128u) + part * (R * 128u) + (k & 3u) * 32u), idesc_s,
                                       part + k > 0);
                        tc_commit(&sh.sfull[b]);
                        if (t + 1 == pc.t1) tc_commit(&sh.qempty[qb]);
                    }
                    __syncwarp();
                    if (n > 0) on = output(n - 1);
                    if (!on) break;
                }
                ++np;
            }
            if (on && n > 0 && !*gave_up) output(n - 1);
        } else if (warp < 4) {
            // ---- queries: a warp per row, split into two e4m3 terms ----
            uint32_t np = 0;
            while (next_piece(a.shape, a.b, shift, walk, &pc)) {
                const uint32_t qb = np & 1u, slot = np % kQSlots;
                if (np >= 2 && !bar_wait(&sh.qempty[qb], ((np >> 1) - 1u) & 1u, gave_up)) break;
                uint8_t* dst = qbuf + qb * C::kQ;
                for (uint32_t r = warp - 2u; r < R; r += 2u) {
                    const uint32_t rr = pc.row_tile * R + r, tok = rr / a.shape.group, g = rr - tok * a.shape.group;
                    const int32_t pos = pc.plan.p0 + static_cast<int32_t>(tok);
                    const bool valid = r < pc.rows;
                    float x[DC][4];
                    float m = 0.0f;
                    bool bad = false;
#pragma unroll
                    for (int c = 0; c < DC; ++c)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t d = c * 128u + lane * 4u + j;
                            x[c][j] = 0.0f;
                            if (valid && d < D) {
                                const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q.data) +
                                                         (pc.plan.row0 + tok) * a.q.token_stride +
                                                         (pc.head * a.shape.group + g) * a.q.head_stride;
                                load_turned<__nv_bfloat16, 1>(a.rope, p, d, pos, &x[c][j]);
                                // a turned query is rounded to its type, as a rotation of its own would
                                x[c][j] = __bfloat162float(__float2bfloat16_rn(x[c][j]));
                            }
                            const float ab = fabsf(x[c][j]);
                            if (ab < __builtin_huge_valf()) m = fmaxf(m, ab);
                            else bad = true;
                        }
                    m = warp_max(m);
                    bad = __any_sync(0xFFFFFFFFu, bad);
                    const int e = kv_scale_exp(m);
                    const float mul = exp2_int(-e);
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const float v0 = x[c][0] * mul, v1 = x[c][1] * mul, v2 = x[c][2] * mul, v3 = x[c][3] * mul;
                        uint32_t h = e4m3x2(v0, v1) | (e4m3x2(v2, v3) << 16);
                        const float2 h01 = e4m3x2_to_float2(h), h23 = e4m3x2_to_float2(h >> 16);
                        uint32_t l = e4m3x2(v0 - h01.x, v1 - h01.y) | (e4m3x2(v2 - h23.x, v3 - h23.y) << 16);
                        if (bad) h = 0x7F7F7F7Fu, l = 0u;  // a NaN or Inf makes the row NaN
                        const uint32_t at = c * (2u * R * 128u) + r * 128u + (((lane >> 2) ^ (r & 7u)) << 4) + (lane & 3u) * 4u;
                        *reinterpret_cast<uint32_t*>(dst + at) = h;
                        *reinterpret_cast<uint32_t*>(dst + at + R * 128u) = l;
                    }
                    if (lane == 0) {
                        sh.frow[slot][r] = exp2_int(e) * (a.scale * kLog2e);
                        sh.qpos[slot][r] = valid ? pos : (-2147483647 - 1);
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    bar_arrive(&sh.qfull[qb]);
                    bar_arrive(&sh.rfull[slot]);
                }
                ++np;
            }
        } else if (warp < 8) {
            // ---- output sums: thread d of a chunk holds element d of every row ----
            const uint32_t quad = warp & 3u, d0 = quad * 32u + lane;
            const uint32_t t_lane = tmem + ((quad * 32u) << 16) + 2u * R;
            uint32_t n = 0, np = 0, meets = 0;
            bool on = true;
            while (on && next_piece(a.shape, a.b, shift, walk, &pc)) {
                float acc[DC][R];
#pragma unroll
                for (int c = 0; c < DC; ++c)
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[c][r] = 0.0f;
                for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                    const uint32_t b = n & 1u;
                    // (the weights' barrier, long complete, orders the factors that the softmax wrote)
                    if (!bar_wait(&sh.ofull[b], (n >> 1) & 1u, gave_up) || !bar_wait(&sh.wfull[b], (n >> 1) & 1u, gave_up)) {
                        on = false;
                        break;
                    }
                    tc_after();
                    const bool changed = (sh.changed[b][0] | sh.changed[b][C::kGroups - 1]) != 0u;
#pragma unroll
                    for (int r = 0; r < R; r += 8) {
                        if (static_cast<uint32_t>(r) >= pc.rows) break;
                        float o[DC][8], o_lo[DC][8];
#pragma unroll
                        for (int c = 0; c < DC; ++c) {
                            tmem_ld8(t_lane + (b * DC + c) * 2u * R + r, o[c]);
                            tmem_ld8(t_lane + (b * DC + c) * 2u * R + R + r, o_lo[c]);
                        }
                        tmem_wait_ld();
                        if (changed) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float al = sh.alpha[b][r + j];
#pragma unroll
                                for (int c = 0; c < DC; ++c) acc[c][r + j] *= al;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float f = sh.osc[b][r + j];
#pragma unroll
                            for (int c = 0; c < DC; ++c)
                                acc[c][r + j] = fmaf(fmaf(o_lo[c][j], kLoInv, o[c][j]), f, acc[c][r + j]);
                        }
                    }
                    tc_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.oempty[b]);
                }
                if (!on || !bar_wait(&sh.lfull, np & 1u, gave_up)) {
                    on = false;
                    break;
                }
                const bool whole = pc.t0 == pc.first && pc.t1 == pc.end;
                const uint32_t r_base = pc.row_tile * R, group = a.shape.group;
                const uint32_t q_heads = a.shape.n_heads * group;
                float* part = a.part + (2ull * blockIdx.x + (pc.t0 == pc.first ? 1u : 0u)) * a.part_stride;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (static_cast<uint32_t>(r) >= pc.rows) break;
                    const float l = sh.lsum[0][r] + sh.lsum[1][r] + sh.lsum[2][r] + sh.lsum[3][r];
                    if (whole) {
                        const uint32_t tok = (r_base + r) / group, g = (r_base + r) - tok * group;
                        __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.out.data) + (pc.plan.row0 + tok) * a.out.token_stride +
                                           (pc.head * group + g) * a.out.head_stride;
                        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                        for (int c = 0; c < DC; ++c)
                            if (c * 128u + d0 < D)
                                p[c * 128u + d0] = __float2bfloat16_rn(l == 0.0f ? 0.0f : acc[c][r] * inv);
                        if (a.lse && d0 == 0u)
                            a.lse[(pc.plan.row0 + tok) * q_heads + pc.head * group + g] = (sh.mfin[r] + log2f(l)) * kLn2;
                    } else {
#pragma unroll
                        for (int c = 0; c < DC; ++c)
                            if (c * 128u + d0 < D) part[r * D + c * 128u + d0] = acc[c][r];
                        if (d0 == 0u) {
                            part[kPartRows * D + r] = sh.mfin[r];
                            part[kPartRows * (D + 1u) + r] = l;
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.lempty);
                ++np;
                if (whole) continue;
                // pieces of one unit meet: the last CTA to arrive joins them in CTA order
                const uint32_t c0 = place_owner(pc.start, total, ctas);
                const uint32_t c1 = place_owner(pc.start + static_cast<uint64_t>(pc.end - pc.first) - 1u, total, ctas);
                __threadfence();
                on = warps_meet(&sh.meet[2], &meets, gave_up);
                if (!on) break;
                if (warp == 4 && lane == 0) {
                    sh.last_flag = atomicAdd(a.counter + c0, 1u) == c1 - c0 ? 1u : 0u;
                    if (sh.last_flag) a.counter[c0] = 0u;
                }
                on = warps_meet(&sh.meet[2], &meets, gave_up);
                if (!on) break;
                if (!sh.last_flag) continue;
                __threadfence();
                for (uint32_t r = 0; r < pc.rows; ++r) {
                    float M = kNegInf, l = 0.0f, o[DC];
#pragma unroll
                    for (int c = 0; c < DC; ++c) o[c] = 0.0f;
                    for (uint32_t c = c0; c <= c1; ++c)
                        M = fmaxf(M, __ldcg(a.part + (2ull * c + (c == c0 ? 1u : 0u)) * a.part_stride + kPartRows * D + r));
                    for (uint32_t c = c0; c <= c1; ++c) {
                        const float* p = a.part + (2ull * c + (c == c0 ? 1u : 0u)) * a.part_stride;
                        const float m = __ldcg(p + kPartRows * D + r);
                        const float f = m == M ? 1.0f : exp2f(m - M);
                        l += __ldcg(p + kPartRows * (D + 1u) + r) * f;
#pragma unroll
                        for (int k = 0; k < DC; ++k)
                            if (k * 128u + d0 < D) o[k] += __ldcg(p + r * D + k * 128u + d0) * f;
                    }
                    const uint32_t tok = (r_base + r) / group, g = (r_base + r) - tok * group;
                    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.out.data) + (pc.plan.row0 + tok) * a.out.token_stride +
                                       (pc.head * group + g) * a.out.head_stride;
#pragma unroll
                    for (int k = 0; k < DC; ++k)
                        if (k * 128u + d0 < D) p[k * 128u + d0] = __float2bfloat16_rn(l == 0.0f ? 0.0f : o[k] / l);
                    if (a.lse && d0 == 0u)
                        a.lse[(pc.plan.row0 + tok) * q_heads + pc.head * group + g] = (M + log2f(l)) * kLn2;
                }
            }
        } else {
            // ---- softmax: a thread per token, its warpgroup's kCols rows ----
            constexpr int NC = C::kCols;
            const uint32_t quad = warp & 3u, grp = (warp - 8u) >> 2, tl = quad * 32u + lane, col0 = grp * NC;
            const uint32_t t_lane = tmem + ((quad * 32u) << 16) + col0;
            float2* my_ref = sh.ref[warp - 8u];
            uint32_t n = 0, np = 0, meets = 0;
            bool on = true;
            while (on && next_piece(a.shape, a.b, shift, walk, &pc)) {
                const uint32_t slot = np % kQSlots;
                if (!bar_wait(&sh.rfull[slot], (np / kQSlots) & 1u, gave_up)) break;
                const float* frow = sh.frow[slot] + col0;
                const int32_t* qpos = sh.qpos[slot] + col0;
                const uint32_t cols = pc.rows > col0 ? min(pc.rows - col0, static_cast<uint32_t>(NC)) : 0u;
                // tiles in [safe0, safe1) are inside every row's positions
                const int32_t p_first = pc.plan.p0 + static_cast<int32_t>(pc.row_tile * R / a.shape.group);
                const int32_t p_last = pc.plan.p0 + static_cast<int32_t>((pc.row_tile * R + pc.rows - 1u) / a.shape.group);
                const int32_t reach = a.shape.all ? pc.plan.len : min(pc.plan.len, p_first + 1);
                const int32_t safe_from = a.shape.window ? p_last - static_cast<int32_t>(a.shape.window) + 1 : 0;
                float l[NC];
#pragma unroll
                for (int c = 0; c < NC; ++c) l[c] = 0.0f;
                float M = kNegInf;  // of row `lane`
                for (int32_t t = pc.t0; t < pc.t1; ++t, ++n) {
                    const uint32_t st = n % NS, b = n & 1u;
                    on = bar_wait(&sh.kfull[st], (n / NS) & 1u, gave_up) && bar_wait(&sh.sfull[b], (n >> 1) & 1u, gave_up);
                    if (!on) break;
                    tc_after();
                    float x[NC];
#pragma unroll
                    for (int c = 0; c < NC; c += 8)
                        if (static_cast<uint32_t>(c) < cols) tmem_ld8(t_lane + b * R + c, x + c);
                    tmem_wait_ld();
                    tc_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.sempty[b]);
                    const int32_t pos = t * kTile + static_cast<int32_t>(tl);
                    const uint32_t pg = tl >> shift;
                    const float fk = sh.kscale[st][pg];
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        if (static_cast<uint32_t>(c & ~7) < cols) x[c] *= fk * frow[c];
                    if (t * kTile < safe_from || (t + 1) * kTile > reach) {
                        const int32_t w = static_cast<int32_t>(a.shape.window);
#pragma unroll
                        for (int c = 0; c < NC; ++c)
                            if (static_cast<uint32_t>(c & ~7) < cols) {
                                const int32_t qp = qpos[c];
                                bool ok = pos < pc.plan.len && (a.shape.all || pos <= qp);
                                if (w) ok = ok && pos > qp - w;
                                if (!ok) x[c] = kNegInf;
                            }
                    }
                    // exponents of the values' scales, relative to the tile's largest: they go into the weights.
                    // Where they differ by much, the weights' factor has to come from the largest product of
                    // weight and scale: the largest weight's own value could be below others' rounding.
                    const int ep = lane < args.pages_per_tile ? scale_exp_of(sh.vscale[st][lane & 7u]) : -127;
                    const int er = __reduce_max_sync(0xFFFFFFFFu, ep);
                    const bool wide = __any_sync(0xFFFFFFFFu, ep > -127 && ep < er - 4);
                    const int ev = scale_exp_of(sh.vscale[st][pg]);
                    const float vr = exp2_int(max(ev - er, -126));
                    // the tile's maximum of every row: lane c ends with row c's
                    float mine = kNegInf;
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        if (static_cast<uint32_t>(c & ~7) < cols) {
                            const float m = warp_max(x[c]);
                            if (lane == static_cast<uint32_t>(c)) mine = m;
                        }
                    if (lane < NC) sh.wmax[b][grp][quad][lane] = mine;
                    if (wide) {  // see below: the largest weight times scale, too
                        float mine2 = kNegInf;
#pragma unroll
                        for (int c = 0; c < NC; ++c)
                            if (static_cast<uint32_t>(c & ~7) < cols) {
                                const float m = warp_max(x[c] + static_cast<float>(max(ev - er, -126)));
                                if (lane == static_cast<uint32_t>(c)) mine2 = m;
                            }
                        if (lane < NC) sh.wmax2[grp][quad][lane] = mine2;
                    }
                    on = warps_meet(&sh.meet[grp], &meets, gave_up);
                    if (!on) break;
                    float mt = kNegInf;
                    if (lane < NC) {
                        mt = fmaxf(fmaxf(sh.wmax[b][grp][0][lane], sh.wmax[b][grp][1][lane]),
                                   fmaxf(sh.wmax[b][grp][2][lane], sh.wmax[b][grp][3][lane]));
                    }
                    const float m1 = fmaxf(M, mt);
                    const float alpha = M == m1 ? 1.0f : ex2(M - m1);
                    // weights e^(x - m1) times 2^(k + 8), k such that the tile's largest is in (128, 256]
                    if (wide) {
                        if (lane < NC)
                            mt = fmaxf(fmaxf(sh.wmax2[grp][0][lane], sh.wmax2[grp][1][lane]),
                                       fmaxf(sh.wmax2[grp][2][lane], sh.wmax2[grp][3][lane]));
                        on = warps_meet(&sh.meet[grp], &meets, gave_up);
                        if (!on) break;
                    }
                    const float gap = m1 - mt;
                    const int k = gap < 100.0f ? static_cast<int>(gap) : (mt == kNegInf ? 0 : 100);
                    __syncwarp();
                    if (lane < NC) my_ref[lane] = make_float2(m1 == kNegInf ? 0.0f : m1, exp2_int(k + 8));
                    const bool changed = __any_sync(0xFFFFFFFFu, alpha != 1.0f);
                    if (quad == 0) {
                        if (n >= 2 && !bar_wait(&sh.oempty[b], ((n >> 1) - 1u) & 1u, gave_up)) {
                            on = false;
                        } else {
                            if (lane < NC) {
                                sh.osc[b][col0 + lane] = exp2_int(max(er, -126)) * exp2_int(-k - 8);
                                sh.alpha[b][col0 + lane] = alpha;
                            }
                            if (lane == 0) sh.changed[b][grp] = changed ? 1u : 0u;
                        }
                    }
                    if (changed) {
#pragma unroll
                        for (int c = 0; c < NC; ++c) l[c] *= __shfl_sync(0xFFFFFFFFu, alpha, c);
                    }
                    M = m1;
                    __syncwarp();
                    if (on && n >= 2) on = bar_wait(&sh.ofull[b], ((n >> 1) - 1u) & 1u, gave_up);  // the weights' buffer
                    if (!on) break;
                    uint8_t* w0 = wbuf + b * C::kW + (tl >> 3) * 128u + (tl & 7u) * 16u;
#pragma unroll
                    for (int c = 0; c < NC; c += 8) {
                        if (static_cast<uint32_t>(c) >= cols) break;
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const float2 r0 = my_ref[c + j], r1 = my_ref[c + j + 1];
                            const float p0 = ex2(x[c + j] - r0.x), p1 = ex2(x[c + j + 1] - r1.x);
                            l[c + j] += p0;
                            l[c + j + 1] += p1;
                            split2(p0 * (r0.y * vr), p1 * (r1.y * vr), &hi[j / 2], &lo[j / 2]);
                        }
                        const uint32_t col = col0 + c;
                        uint8_t* wp = w0 + (col >> 4) * (16u * kTile) + (col & 8u);
                        *reinterpret_cast<uint2*>(wp) = make_uint2(hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16));
                        *reinterpret_cast<uint2*>(wp + R * kTile) = make_uint2(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16));
                    }
                    if ((t + 1) * kTile > pc.plan.len && grp == 0) {
                        // what lies behind the sequence's end may hold NaN bytes, and 0 * NaN is NaN
                        on = bar_wait(&sh.vfull[st], (n / NS) & 1u, gave_up);
                        if (!on) break;
                        if (pos >= pc.plan.len) {
                            uint8_t* v = stages + st * C::kStage + DC * C::kChunk + tl * 128u;
#pragma unroll
                            for (int c = 0; c < DC; ++c)
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    *reinterpret_cast<uint4*>(v + c * C::kChunk + j * 16) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.wfull[b]);
                }
                if (!on) break;
                // the rows' sums over the warp's tokens: lane c ends with row c's
                float mine = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    if (static_cast<uint32_t>(c & ~7) >= cols) continue;
                    float s = l[c];
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
                    if (lane == static_cast<uint32_t>(c)) mine = s;
                }
                if (np >= 1 && !bar_wait(&sh.lempty, (np - 1u) & 1u, gave_up)) break;
                if (lane < NC) {
                    sh.lsum[quad][col0 + lane] = mine;
                    if (quad == 0) sh.mfin[col0 + lane] = M;
                }
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.lfull);
                ++np;
            }
        }
    }
    if (warp == 2 || warp == 3) {
        // statuses: a sequence per warp, over the grid
        for (uint32_t s = blockIdx.x * 2u + (warp - 2u); s < a.b.n_seqs; s += gridDim.x * 2u) {
            const bool ok = seq_pages_ok(a.shape, a.b, shift, a.g.n_pages, s, lane, 32u);
            const bool bad = __any_sync(0xFFFFFFFFu, !ok);
            if (lane == 0) a.status[s] = bad ? SIXI_OUT_OF_BOUNDS : SIXI_OK;
            __syncwarp();
        }
    }

    tc_before();
    __syncthreads();
    tc_after();
    if (sh.gave_up) {
        // never expected: the products in flight end (bounded) before their memory is given back
        if (warp == 1) {
            if (lane == 0) {
                tc_commit(&sh.done);
                for (uint32_t w = 0; w < kWaitIters && !bar_try(&sh.done, 0u); ++w) {}
            }
            __syncwarp();
        }
        for (uint32_t s = tid; s < a.b.n_seqs; s += C::kThreads) a.status[s] = SIXI_BACKEND_ERROR;
    }
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
}

template <int R, int DC>
cudaError_t launch(const MmaArgs& m, const CUtensorMap& k, const CUtensorMap& v, uint32_t n_sms, cudaStream_t stream) {
    using C = Cfg<R, DC>;
    static std::atomic<uint64_t> ready{0};  // the shared-memory opt-in is set once per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(attend_mma_kernel<R, DC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(C::kDyn));
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_acq_rel);
    }
    const uint32_t ctas = n_sms < kAttnMaxCtas ? n_sms : kAttnMaxCtas;
    MmaArgs args = m;
    args.a.shape.rt = R;
    args.a.shape.tile_shift = kTileShift;
    attend_mma_kernel<R, DC><<<ctas, C::kThreads, C::kDyn, stream>>>(args, k, v);
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
    const uint64_t rows = static_cast<uint64_t>(max_new ? max_new : 1u) * a.shape.group;
    if (a.g.head_dim <= 128) {
        if (rows <= 16) return launch<16, 1>(m, k_map, v_map, n_sms, stream);
        if (rows <= 32) return launch<32, 1>(m, k_map, v_map, n_sms, stream);
        return launch<64, 1>(m, k_map, v_map, n_sms, stream);
    }
    if (rows <= 16) return launch<16, 2>(m, k_map, v_map, n_sms, stream);
    return launch<32, 2>(m, k_map, v_map, n_sms, stream);
}

}  // namespace sixi_b200
