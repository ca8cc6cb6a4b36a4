// smp_kv_attn.cu - attention over the 8-bit paged cache in fp32 on the CUDA cores (sixi_kv_attend with
// fp32 queries).
//
// One pass over the cached bytes with the running maximum and sum of a softmax. A CTA works on up to 16
// query rows of one key head at a time (the query heads that share it, times new tokens), so a cached
// byte is brought in once for all of them; 64-token tiles of keys and values are double-buffered in
// shared memory by 16-byte asynchronous copies and widened to fp32 where they are used. Scores: a thread
// takes one token and four rows; values: four elements of a head and every groups-th token.
//
// The work is cut over two CTAs per SM as smp_kv.cuh describes. fp32 products have no tensor-core form that
// keeps 24 bits, so the bound is the fp32 pipes and the shared-memory reads that feed them, and for small
// calls what a piece costs whatever its length: a call of one tile takes 17 us, a further tile of a piece 6, and
// joining 47 pieces some 20. 15 tokens of 6 sequences, up to 3,000 cached ones, 21 heads of 80 elements on 3, cut
// into pieces of one or two tiles: 40 us (the bytes alone would take 0.4 us at the copy rate).
#include <cuda_runtime.h>

#include "smp_kernels.cuh"
#include "smp_kv.cuh"

namespace sixi_b200 {
namespace {

constexpr int kNT = 256;
constexpr int kRt = 16;         // rows of a row tile
constexpr int kTileShift = 6;   // 64 tokens
constexpr int kT = 1 << kTileShift;
constexpr uint32_t kWindow = 32;  // tiles whose page ids are kept
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool on) {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
    const uint32_t n = on ? 16u : 0u;  // 0: the destination is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}

struct Smem {
    float* q;       // [kRt][D], a row divided by a power of two
    uint8_t* kv;    // [2 stages][2][kT][D + 16]
    float* tok;     // [2 stages][2][kT] scales of the tile's tokens
    float* s;       // [kRt][kT]
    float* p;       // [kT][kRt]
    float* alpha;   // [kRt]
    float* m;       // [kRt] running maximum, base 2
    float* l;       // [kRt] running sum
    float* red;     // [4096] sums over token groups
};

// The page ids of tiles [tile, tile + kWindow) of a piece; -1 for pages behind the sequence or before lo's.
__device__ __forceinline__ void load_ids(const AttnArgs& a, const Piece& pc, int32_t lo, int32_t tile, int32_t* ids) {
    const uint32_t per = max(kT >> a.g.page_shift, 1u), shift = a.g.page_shift;
    for (uint32_t i = threadIdx.x; i < kWindow * per; i += kNT) {
        const int32_t pos = (tile << kTileShift) + static_cast<int32_t>(per > 1u ? i << shift : i << kTileShift);
        const uint32_t pg = static_cast<uint32_t>(pos) >> shift;
        const bool on = pos < pc.plan.len && (lo <= 0 || pg >= static_cast<uint32_t>(lo) >> shift);
        ids[i] = on ? a.b.page_table[pc.seq * a.b.table_stride + pg] : -1;
    }
}

// One tile's bytes and scales into stage st; tokens outside the sequence, before the window of the unit's
// first row (lo) or in a bad page are zero.
__device__ __forceinline__ void load_tile(const AttnArgs& a, const Smem& sm, const Piece& pc, int32_t lo, int32_t tile,
                                          uint32_t st, const int32_t* ids) {
    const uint32_t D = a.g.head_dim, row = D + 16u, per = D / 16u, shift = a.g.page_shift;
    uint8_t* dst = sm.kv + static_cast<uint64_t>(st) * 2u * kT * row;
    const uint32_t ids_per = max(kT >> shift, 1u);
    const auto place = [&](uint32_t t, uint64_t* ph) {  // of the tile's token t: its page and head, if it is read
        const int32_t pos = tile * kT + static_cast<int32_t>(t);
        const int32_t id = ids[ids_per > 1u ? t >> shift : 0u];
        *ph = static_cast<uint64_t>(static_cast<uint32_t>(id)) * a.g.n_heads + pc.head;
        return pos < pc.plan.len && pos >= lo && static_cast<uint32_t>(id) < a.g.n_pages;
    };
    for (uint32_t i = threadIdx.x; i < 2u * kT * per; i += kNT) {
        const uint32_t kv = i / (kT * per), j = i - kv * (kT * per);
        const uint32_t t = j / per, c = j - t * per;
        uint64_t ph;
        const bool on = place(t, &ph);
        const uint64_t off =
            on ? (ph * a.g.page_size + (static_cast<uint32_t>(tile * kT + t) & (a.g.page_size - 1u))) * D + c * 16u : 0u;
        cp_async16(dst + (kv * kT + t) * row + c * 16u, (kv ? a.g.v_pages : a.g.k_pages) + off, on);
    }
    if (threadIdx.x < 2u * kT) {
        const uint32_t kv = threadIdx.x >> kTileShift, t = threadIdx.x & (kT - 1u);
        uint64_t ph;
        const bool on = place(t, &ph);
        const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(sm.tok + (st * 2u + kv) * kT + t)), n = on ? 4u : 0u;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"((kv ? a.g.v_scales : a.g.k_scales) + (on ? ph : 0u)),
                     "r"(n)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

__global__ void __launch_bounds__(kNT, 2) attend_f32_kernel(AttnArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ unsigned long long scratch[kNT / 32 + 2];
    __shared__ SeqPlan found;
    __shared__ uint32_t last_flag, disorder;
    __shared__ int32_t ids[kWindow * 4];
    __shared__ uint32_t code[kRt];  // of score_factor
    const uint32_t tid = threadIdx.x, D = a.g.head_dim, row = D + 16u;
    Smem sm;
    {
        float* f = reinterpret_cast<float*>(raw);
        sm.q = f, f += kRt * D;
        sm.kv = reinterpret_cast<uint8_t*>(f), f += 4u * kT * row / 4u;
        sm.tok = f, f += 4 * kT;
        sm.s = f, f += kRt * kT;
        sm.p = f, f += kT * kRt;
        sm.red = f, f += 4096;
        sm.alpha = f, f += kRt;
        sm.m = f, f += kRt;
        sm.l = f;
    }
    if (tid == 0) disorder = 0u;
    PieceWalk walk;
    uint64_t total;
    uint32_t ctas;
    const bool busy = walk_init<kNT>(a.shape, a.b, a.g.page_shift, scratch, &found, &disorder, &walk, &total, &ctas);
    for (uint32_t s = blockIdx.x; s < a.b.n_seqs; s += gridDim.x) {
        const bool ok = disorder == 0u && seq_pages_ok(a.shape, a.b, a.g.page_shift, a.g.n_pages, s, tid, kNT);
        const bool bad = __syncthreads_or(ok ? 0 : 1) != 0;
        if (tid == 0) a.status[s] = a.counter[kAttnMaxCtas] ? SIXI_BACKEND_ERROR : (bad ? SIXI_OUT_OF_BOUNDS : SIXI_OK);
    }
    if (!busy) return;

    const uint32_t quads = D / 4u, groups = kNT / quads;
    const uint32_t quad = tid % quads, tg = tid / quads;
    Piece pc;
    while (next_piece(a.shape, a.b, a.g.page_shift, walk, &pc)) {
        const uint32_t r_base = pc.row_tile * kRt;
        __syncthreads();
        const int32_t lo = a.shape.window ? pc.plan.p0 + static_cast<int32_t>(r_base / a.shape.group) -
                                                static_cast<int32_t>(a.shape.window) + 1
                                          : 0;
        const uint32_t ids_per = max(kT >> a.g.page_shift, 1u);
        load_ids(a, pc, lo, pc.t0, ids);
        __syncthreads();
        load_tile(a, sm, pc, lo, pc.t0, 0, ids);
        // Queries, a warp a row: turned, then divided by a power of two, which keeps their products with the cached bytes
        // within fp32's range. A NaN or Inf makes the row NaN.
        for (uint32_t r = tid >> 5; r < kRt; r += kNT / 32) {
            const uint32_t lane = tid & 31u, tok = (r_base + r) / a.shape.group, g = (r_base + r) - tok * a.shape.group;
            const float* p = static_cast<const float*>(a.q.data) + (pc.plan.row0 + tok) * a.q.token_stride +
                             (pc.head * a.shape.group + g) * a.q.head_stride;
            float m = 0.0f;
            for (uint32_t d = lane; d < D; d += 32u) {
                float x = 0.0f;
                if (r < pc.rows) load_turned<float, 1>(a.rope, p, d, pc.plan.p0 + static_cast<int32_t>(tok), &x);
                m = fabsf(x) < __builtin_huge_valf() ? fmaxf(m, fabsf(x)) : __builtin_huge_valf();
                sm.q[r * D + d] = x;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const bool bad = m == __builtin_huge_valf();
            const int e = bad ? 0 : kv_scale_exp(m);
            const float mul = bad ? __uint_as_float(0x7FC00000u) : exp2_int(-e) * a.score.sign;
            for (uint32_t d = lane; d < D; d += 32u) sm.q[r * D + d] *= mul;
            if (lane == 0) code[r] = score_code(a.score, e);
        }
        if (tid < kRt) sm.m[tid] = kNegInf, sm.l[tid] = 0.0f;
        float acc[kRt][4];
#pragma unroll
        for (int r = 0; r < kRt; ++r) acc[r][0] = acc[r][1] = acc[r][2] = acc[r][3] = 0.0f;

        for (int32_t tile = pc.t0; tile < pc.t1; ++tile) {
            const uint32_t st = static_cast<uint32_t>(tile - pc.t0) & 1u;
            if (tile + 1 < pc.t1) {
                const uint32_t at = static_cast<uint32_t>(tile + 1 - pc.t0) % kWindow;
                if (at == 0) {
                    load_ids(a, pc, lo, tile + 1, ids);
                    __syncthreads();
                }
                load_tile(a, sm, pc, lo, tile + 1, st ^ 1u, ids + at * ids_per);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncthreads();
            const uint8_t* kt = sm.kv + static_cast<uint64_t>(st) * 2u * kT * row;
            const uint8_t* vt = kt + kT * row;
            {  // scores: a thread takes one token and four rows
                const uint32_t t = tid & (kT - 1u), r0 = (tid >> kTileShift) * 4u;
                if (r0 < pc.rows) {
                    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (uint32_t c = 0; c < D; c += 16u) {
                        const uint4 w = *reinterpret_cast<const uint4*>(kt + t * row + c);
                        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 lo = e4m3x2_to_float2(ww[j]), hi = e4m3x2_to_float2(ww[j] >> 16);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float4 q = *reinterpret_cast<const float4*>(sm.q + (r0 + r) * D + c + 4 * j);
                                s[r] = fmaf(q.x, lo.x, fmaf(q.y, lo.y, fmaf(q.z, hi.x, fmaf(q.w, hi.y, s[r]))));
                            }
                        }
                    }
                    const int32_t pos = tile * kT + static_cast<int32_t>(t);
                    const int ek = scale_exp_of(sm.tok[st * 2u * kT + t]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int32_t qp = pc.plan.p0 + static_cast<int32_t>((r_base + r0 + r) / a.shape.group);
                        bool on = pos < pc.plan.len && (a.shape.all || pos <= qp);
                        if (a.shape.window) on = on && pos > qp - static_cast<int32_t>(a.shape.window);
                        sm.s[(r0 + r) * kT + t] = on ? s[r] * score_factor(code[r0 + r], ek) : kNegInf;
                    }
                }
            }
            __syncthreads();
            {  // softmax: a warp takes rows w and w + 8
                const uint32_t lane = tid & 31u;
                const float* vs = sm.tok + (st * 2u + 1u) * kT;
                for (uint32_t r = tid >> 5; r < kRt; r += kNT / 32) {
                    if (r >= pc.rows) {
                        sm.p[lane * kRt + r] = 0.0f;
                        sm.p[(lane + 32u) * kRt + r] = 0.0f;
                        if (lane == 0) sm.alpha[r] = 1.0f;
                        continue;
                    }
                    const float s0 = sm.s[r * kT + lane], s1 = sm.s[r * kT + lane + 32u];
                    float mx = fmaxf(s0, s1);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
                    const float m0 = sm.m[r], m1 = fmaxf(m0, mx);
                    const float p0 = s0 == kNegInf ? 0.0f : exp2f(s0 - m1);
                    const float p1 = s1 == kNegInf ? 0.0f : exp2f(s1 - m1);
                    float sum = p0 + p1;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                    sm.p[lane * kRt + r] = p0 * vs[lane];
                    sm.p[(lane + 32u) * kRt + r] = p1 * vs[lane + 32u];
                    __syncwarp();
                    if (lane == 0) {
                        const float al = m0 == m1 ? 1.0f : exp2f(m0 - m1);
                        sm.alpha[r] = al;
                        sm.m[r] = m1;
                        sm.l[r] = sm.l[r] * al + sum;
                    }
                }
            }
            __syncthreads();
            if (tg < groups) {  // values: a thread takes four elements of a head and every groups-th token
#pragma unroll
                for (int r = 0; r < kRt; ++r) {
                    const float al = sm.alpha[r];
                    acc[r][0] *= al, acc[r][1] *= al, acc[r][2] *= al, acc[r][3] *= al;
                }
                for (uint32_t t = tg; t < kT; t += groups) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(vt + t * row + quad * 4u);
                    const float2 lo = e4m3x2_to_float2(w), hi = e4m3x2_to_float2(w >> 16);
#pragma unroll
                    for (int rb = 0; rb < kRt; rb += 4) {
                        if (static_cast<uint32_t>(rb) >= pc.rows) break;
                        const float4 p = *reinterpret_cast<const float4*>(sm.p + t * kRt + rb);
                        const float pp[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            acc[rb + r][0] = fmaf(pp[r], lo.x, acc[rb + r][0]);
                            acc[rb + r][1] = fmaf(pp[r], lo.y, acc[rb + r][1]);
                            acc[rb + r][2] = fmaf(pp[r], hi.x, acc[rb + r][2]);
                            acc[rb + r][3] = fmaf(pp[r], hi.y, acc[rb + r][3]);
                        }
                    }
                }
            }
            __syncthreads();
        }

        // the piece's sums, four rows at a time over the token groups; whole units go out, others to
        // their partial result
        const bool whole = pc.t0 == pc.first && pc.t1 == pc.end;
        float* part = a.part + (2ull * blockIdx.x + (pc.t0 == pc.first ? 1u : 0u)) * a.part_stride;
#pragma unroll
        for (int rb = 0; rb < kRt; rb += 4) {
            if (static_cast<uint32_t>(rb) >= pc.rows) break;
            __syncthreads();
            if (tg < groups) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    *reinterpret_cast<float4*>(sm.red + ((tg * 4u + r) * quads + quad) * 4u) =
                        make_float4(acc[rb + r][0], acc[rb + r][1], acc[rb + r][2], acc[rb + r][3]);
            }
            __syncthreads();
            for (uint32_t i = tid; i < 4u * D; i += kNT) {
                const uint32_t r = i / D, d = i - r * D;
                if (rb + r >= pc.rows) continue;
                float o = 0.0f;
                for (uint32_t g = 0; g < groups; ++g) o += sm.red[(g * 4u + r) * D + d];
                if (whole) {
                    const uint32_t rr = r_base + rb + r, tok = rr / a.shape.group, g = rr - tok * a.shape.group;
                    const float l = sm.l[rb + r];
                    float* p = static_cast<float*>(a.out.data) + (pc.plan.row0 + tok) * a.out.token_stride +
                           (pc.head * a.shape.group + g) * a.out.head_stride + d;
                    *p = l == 0.0f ? 0.0f : o / l;
                } else {
                    part[(rb + r) * D + d] = o;
                }
            }
        }
        if (tid < pc.rows) {
            if (whole) {
                if (a.lse) {
                    const uint32_t rr = r_base + tid, tok = rr / a.shape.group, g = rr - tok * a.shape.group;
                    a.lse[(pc.plan.row0 + tok) * (a.shape.n_heads * a.shape.group) + pc.head * a.shape.group + g] =
                        (sm.m[tid] + log2f(sm.l[tid])) * kLn2;
                }
            } else {
                part[kRt * D + tid] = sm.m[tid];
                part[kRt * (D + 1u) + tid] = sm.l[tid];
            }
        }
        if (whole) continue;
        const uint32_t c0 = place_owner(pc.start, total, ctas);
        const uint32_t c1 = place_owner(pc.start + static_cast<uint64_t>(pc.end - pc.first) - 1u, total, ctas);
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            last_flag = atomicAdd(a.counter + c0, 1u) == c1 - c0 ? 1u : 0u;
            if (last_flag) a.counter[c0] = 0u;
        }
        __syncthreads();
        if (!last_flag) continue;
        __threadfence();
        // the last CTA of the unit joins the pieces
        join_rows<float, 2, 2, 2>(a, a.part + (2ull * c0 + 1u) * a.part_stride, a.part + 2ull * c0 * a.part_stride, c1 - c0 + 1u,
                        pc.rows, r_base, pc.plan.row0, pc.head, tid >> 5);
    }
}

}  // namespace

cudaError_t launch_attend_f32(AttnArgs a, uint32_t n_sms, cudaStream_t stream) {
    a.shape.rt = kRt;
    a.shape.tile_shift = kTileShift;
    a.shape.unit_cost = 2;
    // a tile of a unit takes 6 us and joining its pieces 2 to 4 (2 tokens of 21 heads on 3 of 80 over 250 and 500 cached ones:
    // 19.8 and 21.3 us cut, 34.9 and 58.0 whole; 100 such sequences over 500: 90 and 137)
    a.shape.whole_tiles = 1;
    a.part_stride = part_floats(kRt, a.g.head_dim);
    const uint32_t D = a.g.head_dim;
    const size_t smem = sizeof(float) * (static_cast<size_t>(kRt) * D + 4u * kT * (D + 16u) / 4u + 4u * kT + 2u * kRt * kT +
                                         4096u + 3u * kRt);
    const cudaError_t e = cudaFuncSetAttribute(attend_f32_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    const uint32_t ctas = 2u * n_sms < kAttnMaxCtas ? 2u * n_sms : kAttnMaxCtas;
    attend_f32_kernel<<<ctas, kNT, smem, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace sixi_b200
