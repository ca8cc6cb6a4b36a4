// smp_kv.cu - rotary positions, writing and reading the 8-bit paged key/value cache, and the
// extern "C" boundary of include/sixi_kv.h (attention: smp_kv_attn.cu).
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "smp_device.cuh"
#include "smp_kernels.cuh"
#include "smp_kv.cuh"

namespace sixi_b200 {
namespace {

constexpr int kNT = 256;

// ---------------------------------------------------------------------------------------------
// sixi_kv_rope_apply: (a, b) -> amp * (a cos - b sin, b cos + a sin) for pair i of a head's first rot_dim elements, the
// angle position * f_i; the inverse has the sine's sign turned, which is also the gradient. Bound by memory: every element
// is read and written once. A thread takes VEC pairs (half layout) or VEC / 2 pairs (interleaved) of one token, computes
// their sines once and turns those elements of `hpt` heads; the elements that are passed through are further chunks.
// 16,384 tokens of 40 heads of 128 bf16 elements (half layout): 58.2 us, 5.8 TB/s, 88 % of the copy rate. 5 tokens of 12
// heads: 2.3 us, the launch.

template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kNT) rope_kernel(RopeView r, KvView x, KvView out, const int32_t* __restrict__ positions,
                                                   uint64_t n_items, uint32_t chunks, uint32_t turned, uint32_t n_heads,
                                                   uint32_t hpt, uint32_t hgroups) {
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * kNT + threadIdx.x;
    if (item >= n_items) return;
    const uint64_t th = item / chunks;
    const uint32_t chunk = static_cast<uint32_t>(item - th * chunks);
    const uint64_t token = th / hgroups;
    const uint32_t h0 = static_cast<uint32_t>(th - token * hgroups) * hpt;
    const uint32_t h1 = min(h0 + hpt, n_heads);
    const T* px = static_cast<const T*>(x.data) + token * x.token_stride;
    T* po = static_cast<T*>(out.data) + token * out.token_stride;
    if (chunk >= turned) {  // passed through
        const uint32_t i0 = r.rot_dim + (chunk - turned) * VEC;
        for (uint32_t h = h0; h < h1; ++h) {
            float v[VEC];
            load_vec<T, VEC>(px + h * x.head_stride + i0, v);
            store_vec<T, VEC>(po + h * out.head_stride + i0, v);
        }
        return;
    }
    const int32_t pos = positions[token];
    if constexpr (!INTER) {
        const uint32_t i0 = chunk * VEC, half = r.rot_dim >> 1;
        float s[VEC], c[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) rope_sincos(r, pos, i0 + j, &s[j], &c[j]);
        for (uint32_t h = h0; h < h1; ++h) {
            const T* p = px + h * x.head_stride;
            T* o = po + h * out.head_stride;
            float a[VEC], b[VEC];
            load_vec<T, VEC>(p + i0, a);
            load_vec<T, VEC>(p + i0 + half, b);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float ya = a[j] * c[j] - b[j] * s[j];
                b[j] = b[j] * c[j] + a[j] * s[j];
                a[j] = ya;
            }
            store_vec<T, VEC>(o + i0, a);
            store_vec<T, VEC>(o + i0 + half, b);
        }
    } else {
        constexpr int W = VEC == 1 ? 2 : VEC;  // elements of a chunk
        const uint32_t i0 = chunk * W;
        float s[W / 2], c[W / 2];
#pragma unroll
        for (int j = 0; j < W / 2; ++j) rope_sincos(r, pos, (i0 >> 1) + j, &s[j], &c[j]);
        for (uint32_t h = h0; h < h1; ++h) {
            const T* p = px + h * x.head_stride + i0;
            T* o = po + h * out.head_stride + i0;
            float a[W];
            if constexpr (VEC == 1) {
                load_vec<T, 1>(p, a);
                load_vec<T, 1>(p + 1, a + 1);
            } else {
                load_vec<T, VEC>(p, a);
            }
#pragma unroll
            for (int j = 0; j < W; j += 2) {
                const float u = a[j], v = a[j + 1];
                a[j] = u * c[j / 2] - v * s[j / 2];
                a[j + 1] = v * c[j / 2] + u * s[j / 2];
            }
            if constexpr (VEC == 1) {
                store_vec<T, 1>(o, a);
                store_vec<T, 1>(o + 1, a + 1);
            } else {
                store_vec<T, VEC>(o, a);
            }
        }
    }
}

bool view_aligned(const sixi_kv_tensor* t, uint32_t n_heads, uint32_t n_tokens) {
    const uint64_t esz = t->dtype == SIXI_SMP_BF16 ? 2 : 4;
    return (reinterpret_cast<uintptr_t>(t->data) & 15u) == 0 && (n_heads < 2 || (t->head_stride * esz) % 16 == 0) &&
           (n_tokens < 2 || (t->token_stride * esz) % 16 == 0);
}

KvView view_of(const sixi_kv_tensor* t) { return KvView{t->data, t->token_stride, t->head_stride}; }

template <typename T, int VEC, bool INTER>
cudaError_t rope_launch(const RopeView& r, const sixi_kv_tensor* x, const int32_t* positions, uint32_t n_tokens,
                        uint32_t head_dim, const sixi_kv_tensor* out, cudaStream_t stream) {
    const uint32_t w = INTER ? (VEC == 1 ? 2 : VEC) : 2 * VEC;  // elements that a turned chunk covers
    const uint32_t turned = r.rot_dim / w;
    const bool same = x->data == out->data && x->token_stride == out->token_stride && x->head_stride == out->head_stride;
    const uint32_t chunks = turned + (same ? 0u : (head_dim - r.rot_dim) / VEC);
    const uint32_t heads = x->n_heads;
    // heads per thread: the sines of a chunk are worth sharing once the GPU's threads are all busy
    const uint64_t all = static_cast<uint64_t>(n_tokens) * chunks * heads;
    uint32_t hpt = static_cast<uint32_t>(all / (148ull * 2048ull));
    hpt = hpt < 1 ? 1 : (hpt > 8 ? 8 : hpt);
    if (hpt > heads) hpt = heads;
    const uint32_t hgroups = (heads + hpt - 1) / hpt;
    const uint64_t items = static_cast<uint64_t>(n_tokens) * hgroups * chunks;
    const uint64_t blocks = (items + kNT - 1) / kNT;
    if (blocks == 0) return cudaSuccess;
    if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    rope_kernel<T, VEC, INTER><<<static_cast<uint32_t>(blocks), kNT, 0, stream>>>(
        r, view_of(x), view_of(out), positions, items, chunks, turned, heads, hpt, hgroups);
    return cudaGetLastError();
}

template <typename T, int V>
cudaError_t rope_dispatch(const RopeView& r, const sixi_kv_tensor* x, const int32_t* positions, uint32_t n_tokens,
                          uint32_t head_dim, const sixi_kv_tensor* out, cudaStream_t stream) {
    const bool al = view_aligned(x, x->n_heads, n_tokens) && view_aligned(out, out->n_heads, n_tokens) &&
                    (head_dim - r.rot_dim) % V == 0;
    if (r.interleaved)
        return al && r.rot_dim % V == 0 ? rope_launch<T, V, true>(r, x, positions, n_tokens, head_dim, out, stream)
                                        : rope_launch<T, 1, true>(r, x, positions, n_tokens, head_dim, out, stream);
    return al && (r.rot_dim / 2) % V == 0 ? rope_launch<T, V, false>(r, x, positions, n_tokens, head_dim, out, stream)
                                          : rope_launch<T, 1, false>(r, x, positions, n_tokens, head_dim, out, stream);
}

// ---------------------------------------------------------------------------------------------
// sixi_kv_append. With m the largest magnitude of a page's and head's new rows, e the least exponent with m <= 448 * 2^e
// and e' the page's own: scale 2^max(e, e'), bytes e4m3(x / scale). The scale is a maximum over rows, so a page's rows of
// one head (a unit) are the work of one team, which holds the first kRowsHeld rows of a lane in registers between the
// maximum and the rounding; further ones are read again. A row takes the lanes of D / 8 elements, 8 each.
//
// Bound: a prompt by memory (18,796 tokens of 8 heads of 128 bf16 elements: 116 MB in and out, 17.7 us at the copy rate,
// 55.5 us with the keys' rotation and 38 without, most of it the waits of a CTA's steps: rows, maximum, bytes); few tokens
// by latency: the chain of sequence, page, rows and scale is 4.7 us for 64 tokens of 64 sequences. So:
// - few rows (up to kRowsFew a page): a unit is at most a warp's, and a CTA takes many units. 153 tokens of 37 sequences,
//   9 at most: 6.0 us, and 8.1 with a CTA a unit.
// - many rows: the whole CTA is the team, rows side by side, up to four heads one after the other, which share their
//   tokens' sines (with two heads 62 us with the rotation and 38 without, with eight 54.5 and 45).
// - a page that holds older rows and whose scale grows: all its older rows are rounded again by the whole CTA, whoever's
//   unit it is. It happens to few units at a time: 10.2 us where one head of 16 grows (64 tokens, pages of 64 with 60
//   older rows, memory cold), 22.5 when the unit's team does it alone, 10.2 without growth.
//
// An item is a page that a sequence's new tokens touch. Items are numbered so that the host needs no lengths: sequence s
// starts at floor(offsets[s] / page_size) + 2 s, which leaves room for every page that it can touch.

struct AppendArgs {
    KvGeom g;
    KvBatchView b;
    KvView k, v;
    RopeView rope;
    int32_t* status;
    uint32_t* seq_state;  // [2 * max_seqs]: arrivals, flags; zero between calls
    uint32_t row_lanes;   // lanes of a row: the power of two at or above D / 8
    uint32_t team;        // threads of a team: row_lanes or kNT
    uint32_t heads;       // with a team of kNT: heads of keys, or of values, that a CTA takes one after the other
};

constexpr int kRowsHeld = 4;
constexpr uint32_t kRowsFew = 16;
constexpr size_t kSinesMax = 64u * 1024u;
constexpr uint32_t kFlagNan = 1u, kFlagBounds = 2u;

__device__ __forceinline__ uint32_t item_base(int64_t row0, uint32_t page_shift, uint32_t s) {
    return static_cast<uint32_t>(static_cast<uint64_t>(row0) >> page_shift) + 2u * s;
}

// 8 elements of a row, turned
template <typename T, int VEC>
__device__ __forceinline__ void load_row8(const RopeView& r, const T* p, uint32_t i0, int32_t pos, float* x) {
#pragma unroll
    for (int j = 0; j < 8; j += VEC) load_turned<T, VEC>(r, p, i0 + j, pos, x + j);
}
// 8 elements of a row, as loaded to x, turned with the row's sines at hand (the other halves come from p again)
template <typename T, int VEC>
__device__ __forceinline__ void turn8(const RopeView& r, const T* p, uint32_t i0, const float2* sines, float* x) {
    const uint32_t half = r.rot_dim >> 1;
    if (r.interleaved) {
#pragma unroll
        for (uint32_t j = 0; j < 8; j += 2) {
            if (i0 + j >= r.rot_dim) continue;
            const float2 t = sines[(i0 + j) >> 1];
            const float y = x[j] * t.x - x[j + 1] * t.y;
            x[j + 1] = x[j + 1] * t.x + x[j] * t.y;
            x[j] = y;
        }
    } else if constexpr (VEC == 1) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t i = i0 + j;
            if (i >= r.rot_dim) continue;
            const bool upper = i >= half;
            const float2 t = sines[upper ? i - half : i];
            float o;
            load_vec<T, 1>(p + (upper ? i - half : i + half), &o);
            x[j] = upper ? x[j] * t.x + o * t.y : x[j] * t.x - o * t.y;
        }
    } else if (i0 < r.rot_dim) {
        const bool upper = i0 >= half;
        const uint32_t p0 = upper ? i0 - half : i0;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; j += VEC) load_vec<T, VEC>(p + (upper ? p0 : i0 + half) + j, o + j);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 t = sines[p0 + j];
            x[j] = upper ? x[j] * t.x + o[j] * t.y : x[j] * t.x - o[j] * t.y;
        }
    }
}
// NaN as 0; *m the largest finite magnitude
__device__ __forceinline__ void clean8(float* x, float* m, bool* bad) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float a = fabsf(x[j]);
        if (!(a < __builtin_huge_valf())) {
            *bad = true;
            if (a != a) x[j] = 0.0f;
        } else {
            *m = fmaxf(*m, a);
        }
    }
}

__device__ __forceinline__ void unpack8_e4m3(uint2 o, float* y) {
    float2 f;
    f = e4m3x2_to_float2(o.x), y[0] = f.x, y[1] = f.y;
    f = e4m3x2_to_float2(o.x >> 16), y[2] = f.x, y[3] = f.y;
    f = e4m3x2_to_float2(o.y), y[4] = f.x, y[5] = f.y;
    f = e4m3x2_to_float2(o.y >> 16), y[6] = f.x, y[7] = f.y;
}

__device__ __forceinline__ uint2 round8(const float* x, float mul) {
    uint2 o;
    o.x = e4m3x2(x[0] * mul, x[1] * mul) | (e4m3x2(x[2] * mul, x[3] * mul) << 16);
    o.y = e4m3x2(x[4] * mul, x[5] * mul) | (e4m3x2(x[6] * mul, x[7] * mul) << 16);
    return o;
}

// MODE 0: keys as they are; 1: turned, a CTA's heads sharing their tokens' sines; 2: turned, every lane its own
enum { kAsIs = 0, kSharedSines = 1, kOwnSines = 2 };

template <typename T, int VEC, int MODE>
__global__ void __launch_bounds__(kNT, MODE == kAsIs && VEC > 1 ? 4 : (MODE == kSharedSines && VEC > 1 ? 3 : 2))
    append_kernel(AppendArgs a) {
    __shared__ float red[kNT / 32];
    __shared__ KvSeq item_q;
    __shared__ uint32_t item_seq, item_page;
    __shared__ int32_t item_id;
    __shared__ uint32_t n_grown;
    __shared__ uint8_t* grown_page[kNT / 2];  // (a row has two lanes at least)
    __shared__ float grown_mul[kNT / 2];
    extern __shared__ float2 sines[];  // [new rows of the page][rot_dim / 2], with shared sines
    const uint32_t tid = threadIdx.x;
    if (tid == 0) n_grown = 0u;
    // the sequences whose status needs no pages (no new tokens, or numbers that do not fit)
    if (blockIdx.y == 0 && blockIdx.x < a.b.n_seqs && tid == 0) {
        const KvSeq q = kv_seq(a.b, a.g.page_shift, blockIdx.x);
        const bool ok = q.ok && q.len >= q.n;
        if (!ok || q.n == 0) a.status[blockIdx.x] = ok ? SIXI_OK : SIXI_OUT_OF_BOUNDS;
    }
    // the item's sequence and page: found by the thread that comes upon the sequence, so that a CTA's way to its rows is
    // three loads long
    bool in_order = true, mine = false;
    for (uint32_t s = tid; s < a.b.n_seqs; s += kNT) {
        const int64_t r0 = a.b.offsets[s], r1 = a.b.offsets[s + 1];
        const int32_t len = a.b.lens[s];
        in_order &= r0 >= 0 && r1 >= r0 && r1 <= static_cast<int64_t>(a.b.n_tokens);
        const uint32_t at = item_base(r0, a.g.page_shift, s), next = item_base(r1, a.g.page_shift, s + 1u);
        if (at <= blockIdx.x && (blockIdx.x < next || s + 1u == a.b.n_seqs)) {
            const KvSeq q = kv_seq_of(a.b, a.g.page_shift, r0, r1, len);
            const int32_t start = q.len - q.n;
            const uint32_t pi = (static_cast<uint32_t>(start) >> a.g.page_shift) + (blockIdx.x - at);
            mine = q.ok && q.n > 0 && start >= 0 && pi <= static_cast<uint32_t>(q.len - 1) >> a.g.page_shift;
            if (mine) {
                item_q = q;
                item_seq = s;
                item_page = pi;
                item_id = a.b.page_table[s * a.b.table_stride + pi];
            }
        }
    }
    if (__syncthreads_or(in_order ? 0 : 1)) {  // items cannot be told from one another
        if (blockIdx.y == 0 && blockIdx.x < a.b.n_seqs && tid == 0) a.status[blockIdx.x] = SIXI_OUT_OF_BOUNDS;
        return;
    }
    if (!__syncthreads_or(mine ? 1 : 0)) return;
    const uint32_t seq = item_seq, pi = item_page;
    const KvSeq q = item_q;
    const int32_t start = q.len - q.n;
    const uint32_t first_page = static_cast<uint32_t>(start) >> a.g.page_shift;
    const uint32_t last_page = static_cast<uint32_t>(q.len - 1) >> a.g.page_shift;
    const int32_t page0 = static_cast<int32_t>(pi << a.g.page_shift);
    const uint32_t slot0 = static_cast<uint32_t>(max(start, page0) - page0);
    const uint32_t slot1 = static_cast<uint32_t>(min(q.len - page0, static_cast<int32_t>(a.g.page_size)));
    const int32_t id = item_id;
    const bool id_ok = static_cast<uint32_t>(id) < a.g.n_pages;

    const uint32_t teams = kNT / a.team;
    const uint32_t D = a.g.head_dim;
    const uint32_t in_team = tid % a.team;
    const uint32_t i0 = (in_team % a.row_lanes) * 8u;
    const uint32_t row_in = in_team / a.row_lanes, rows_at_once = a.team / a.row_lanes;
    // units of this CTA: one a team, or those of some heads one after the other
    const uint32_t groups = a.heads ? (a.g.n_heads + a.heads - 1u) / a.heads : 0u;  // of keys, then of values
    const uint32_t half = a.rope.rot_dim >> 1;
    if (MODE == kSharedSines && blockIdx.y < groups && id_ok) {
        for (uint32_t i = tid; i < (slot1 - slot0) * half; i += kNT) {
            const uint32_t r = i / half, p = i - r * half;
            float sn, cs;
            rope_sincos(a.rope, page0 + static_cast<int32_t>(slot0 + r), p, &sn, &cs);
            sines[i] = make_float2(cs, sn);
        }
        __syncthreads();
    }
    uint32_t unit0 = blockIdx.y * teams + tid / a.team, unit_end = unit0 + 1u;
    if (a.heads) {
        const bool values = blockIdx.y >= groups;
        const uint32_t h0 = (blockIdx.y - (values ? groups : 0u)) * a.heads;
        unit0 = (values ? a.g.n_heads : 0u) + h0;
        unit_end = (values ? a.g.n_heads : 0u) + min(h0 + a.heads, a.g.n_heads);
    }
    bool bad = false;
    for (uint32_t unit = unit0; unit < unit_end; ++unit) {
        const bool live = id_ok && unit < 2u * a.g.n_heads;
        const bool is_v = unit >= a.g.n_heads;
        const uint32_t head = is_v ? unit - a.g.n_heads : unit;
        const KvView& src = is_v ? a.v : a.k;
        const bool turn = MODE != kAsIs && !is_v;
        const T* base = static_cast<const T*>(src.data) + head * src.head_stride;
        const bool lane_on = live && i0 < D;
        const auto row_of = [&](uint32_t slot) {
            return base + (q.row0 + (page0 + static_cast<int32_t>(slot) - start)) * src.token_stride;
        };
        const auto turn_row = [&](uint32_t slot, float* y) {  // y: the row's elements as loaded
            if constexpr (MODE == kSharedSines) turn8<T, VEC>(a.rope, row_of(slot), i0, sines + (slot - slot0) * half, y);
            if constexpr (MODE == kOwnSines) load_row8<T, VEC>(a.rope, row_of(slot), i0, page0 + static_cast<int32_t>(slot), y);
        };
        const auto load = [&](uint32_t slot, float* y, float* mm) {
#pragma unroll
            for (int j = 0; j < 8; j += VEC) load_vec<T, VEC>(row_of(slot) + i0 + j, y + j);
            if (turn) turn_row(slot, y);
            clean8(y, mm, &bad);
        };

        float x[kRowsHeld][8];
        float m = 0.0f;
        if (lane_on) {
            // the held rows' elements are asked for together, then worked on
#pragma unroll
            for (int p = 0; p < kRowsHeld; ++p) {
                const uint32_t slot = min(slot0 + p * rows_at_once + row_in, slot1 - 1u);
                const T* r = row_of(slot);
#pragma unroll
                for (int j = 0; j < 8; j += VEC) load_vec<T, VEC>(r + i0 + j, x[p] + j);
            }
#pragma unroll
            for (int p = 0; p < kRowsHeld; ++p) {
                const uint32_t slot = slot0 + p * rows_at_once + row_in;
                if (slot >= slot1) continue;
                if (turn) turn_row(slot, x[p]);
                clean8(x[p], &m, &bad);
            }
            for (uint32_t slot = slot0 + kRowsHeld * rows_at_once + row_in; slot < slot1; slot += rows_at_once) {
                float y[8];
                load(slot, y, &m);
            }
        }
        // the unit's maximum: over the lanes of a row by shuffles, over the CTA's warps through shared memory
        const uint32_t width = a.team < 32u ? a.team : 32u;
        for (uint32_t o = width >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if (a.team > 32u) {
            __syncthreads();  // (the last unit's have been read)
            if ((tid & 31u) == 0) red[tid >> 5] = m;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kNT / 32; ++i) m = fmaxf(m, red[i]);
        }
        float* sp = nullptr;
        int e = 0;
        bool write_scale = false;
        if (live) {
            const uint64_t ph = static_cast<uint64_t>(id) * a.g.n_heads + head;
            sp = (is_v ? a.g.v_scales : a.g.k_scales) + ph;
            uint8_t* pg = (is_v ? a.g.v_pages : a.g.k_pages) + ph * a.g.page_size * D;
            e = kv_scale_exp(m);
            write_scale = true;
            if (slot0 > 0) {
                const int eo = scale_exp_of(*sp);
                if (e > eo) {  // the page's scale grows
                    if (in_team == 0) {
                        const uint32_t g = atomicAdd(&n_grown, 1u);
                        grown_page[g] = pg;
                        grown_mul[g] = exp2_int(max(eo - e, -126));
                    }
                } else {
                    e = eo;
                    write_scale = false;
                }
            }
            const float mul = exp2_int(-e);
            if (lane_on) {
#pragma unroll
                for (int p = 0; p < kRowsHeld; ++p) {
                    const uint32_t slot = slot0 + p * rows_at_once + row_in;
                    if (slot < slot1) *reinterpret_cast<uint2*>(pg + slot * D + i0) = round8(x[p], mul);
                }
                for (uint32_t slot = slot0 + kRowsHeld * rows_at_once + row_in; slot < slot1; slot += rows_at_once) {
                    float y[8], again = 0.0f;
                    load(slot, y, &again);
                    *reinterpret_cast<uint2*>(pg + slot * D + i0) = round8(y, mul);
                }
            }
        }
        // every lane of the team has read the old scale before it is replaced (by all threads of the CTA:
        // lanes without a unit must not miss the barrier)
        __syncthreads();
        if (in_team == 0 && write_scale) *sp = exp2_int(e);
        // The older rows of pages whose scale has grown are rounded again at it, by the whole CTA: they may be a page's worth
        // for a single new token, and seldom of more than one of the CTA's units.
        const uint32_t grown = n_grown;
        if (grown > 0u) {
            const uint32_t per_row = D / 8u, per_page = slot0 * per_row, all = grown * per_page;
            for (uint32_t c0 = tid; c0 < all; c0 += 4u * kNT) {
                uint2* at[4];
                uint2 o[4];
                float mul[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t c = min(c0 + u * kNT, all - 1u), g = c / per_page;
                    at[u] = reinterpret_cast<uint2*>(grown_page[g]) + (c - g * per_page);
                    mul[u] = grown_mul[g];
                    o[u] = *at[u];
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float y[8];
                    unpack8_e4m3(o[u], y);
                    if (c0 + u * kNT < all) *at[u] = round8(y, mul[u]);
                }
            }
            __syncthreads();
            if (tid == 0) n_grown = 0u;  // (the next unit's team meets before it adds to it)
        }
    }
    // the sequence's status: the last of its CTAs to arrive writes it
    const bool any_bad = __syncthreads_or(bad ? 1 : 0) != 0;
    if (tid == 0) {
        const uint32_t flag = (any_bad ? kFlagNan : 0u) | (id_ok ? 0u : kFlagBounds);
        const uint32_t ctas = (last_page - first_page + 1u) * gridDim.y;
        uint32_t flags = flag;
        bool last = true;
        if (ctas > 1u) {
            uint32_t* st = a.seq_state + 2u * seq;
            // (only a raised flag has to be seen before the arrival; the pages themselves need no order here)
            if (flag) {
                atomicOr(st + 1, flag);
                __threadfence();
            }
            last = atomicAdd(st, 1u) == ctas - 1u;
            if (last) {
                __threadfence();
                flags = atomicExch(st + 1, 0u);
                atomicExch(st, 0u);
            }
        }
        if (last)
            a.status[seq] = (flags & kFlagBounds) ? SIXI_OUT_OF_BOUNDS
                                                  : ((flags & kFlagNan) ? SIXI_NUMERIC_NAN_OR_INF : SIXI_OK);
    }
}

// ---------------------------------------------------------------------------------------------
// sixi_kv_read: bytes times scale, 8 elements a lane at a time; a warp takes a token, so that its page is looked up once,
// and keeps four loads in flight. Bound by memory: 18,796 tokens of 8 heads of 128 elements into bf16, keys and values:
// 28.2 us, 4.1 TB/s. A token of each of 64 sequences: 4.7 us, the chain of lookups.

struct ReadArgs {
    KvGeom g;
    KvBatchView b;
    KvView k, v;
    int32_t* status;
    uint32_t per;  // tokens of a CTA
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kNT) read_kernel(ReadArgs a) {
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    const bool in_order = __syncthreads_or(kv_offsets_ok(a.b, tid, kNT) ? 0 : 1) == 0;
    if (blockIdx.y == 0) {  // statuses, spread over the CTAs
        for (uint32_t s = blockIdx.x; s < a.b.n_seqs; s += gridDim.x) {
            const KvSeq q = kv_seq(a.b, a.g.page_shift, s);
            bool bad = !in_order || !q.ok || q.len < q.n;
            if (!bad && q.n > 0) {
                const uint32_t p0 = static_cast<uint32_t>(q.len - q.n) >> a.g.page_shift;
                const uint32_t p1 = static_cast<uint32_t>(q.len - 1) >> a.g.page_shift;
                for (uint32_t p = p0 + tid; p <= p1; p += kNT)
                    bad |= static_cast<uint32_t>(a.b.page_table[s * a.b.table_stride + p]) >= a.g.n_pages;
            }
            bad = __syncthreads_or(bad ? 1 : 0) != 0;
            if (tid == 0) a.status[s] = bad ? SIXI_OUT_OF_BOUNDS : SIXI_OK;
        }
    }
    if (!in_order) return;
    const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * a.per;
    const uint64_t t1 = t0 + a.per < a.b.n_tokens ? t0 + a.per : a.b.n_tokens;
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.b.n_seqs; s0 += kNT) {
        const uint32_t s = s0 + tid;
        before += __syncthreads_count(s < a.b.n_seqs && a.b.offsets[s] <= static_cast<int64_t>(t0));
    }
    if (before == 0) return;
    const bool is_v = blockIdx.y != 0;
    const KvView& dst = is_v ? a.v : a.k;
    const uint8_t* pages = is_v ? a.g.v_pages : a.g.k_pages;
    const float* scales = is_v ? a.g.v_scales : a.g.k_scales;
    const uint32_t D = a.g.head_dim, row_chunks = D / 8u, chunks = a.g.n_heads * row_chunks;
    uint32_t seq = before - 1;
    KvSeq q = kv_seq(a.b, a.g.page_shift, seq);
    for (uint64_t tok = t0 + (tid >> 5); tok < t1; tok += kNT / 32) {
        while (seq + 1 < a.b.n_seqs && a.b.offsets[seq + 1] <= static_cast<int64_t>(tok)) {
            ++seq;
            q = kv_seq(a.b, a.g.page_shift, seq);
        }
        const int64_t in = static_cast<int64_t>(tok) - q.row0;
        if (!q.ok || q.len < q.n || in < 0 || in >= q.n) continue;
        const uint32_t pos = static_cast<uint32_t>(q.len - q.n + static_cast<int32_t>(in));
        const int32_t id = a.b.page_table[seq * a.b.table_stride + (pos >> a.g.page_shift)];
        const bool good = static_cast<uint32_t>(id) < a.g.n_pages;
        const uint64_t ph0 = static_cast<uint64_t>(good ? id : 0) * a.g.n_heads;
        const uint32_t slot = pos & (a.g.page_size - 1u);
        T* out = static_cast<T*>(dst.data) + tok * dst.token_stride;
        constexpr int kUnroll = 4;
        for (uint32_t c0 = lane; c0 < chunks; c0 += 32u * kUnroll) {
            uint2 o[kUnroll];
            float f[kUnroll];
            uint32_t head[kUnroll], i0[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const uint32_t c = min(c0 + 32u * u, chunks - 1u);
                head[u] = c / row_chunks;
                i0[u] = (c - head[u] * row_chunks) * 8u;
                o[u] = make_uint2(0u, 0u);
                f[u] = 0.0f;
                if (good) {
                    o[u] = *reinterpret_cast<const uint2*>(pages + ((ph0 + head[u]) * a.g.page_size + slot) * D + i0[u]);
                    f[u] = scales[ph0 + head[u]];
                }
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (c0 + 32u * u >= chunks) continue;
                float y[8];
                unpack8_e4m3(o[u], y);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] *= f[u];
                T* p = out + head[u] * dst.head_stride + i0[u];
#pragma unroll
                for (int j = 0; j < 8; j += VEC) store_vec<T, VEC>(p + j, y + j);
            }
        }
    }
}

}  // namespace

cudaError_t launch_rope_apply(const RopeView& r, const sixi_kv_tensor* x, const int32_t* positions, uint32_t n_tokens,
                              uint32_t head_dim, const sixi_kv_tensor* out, cudaStream_t stream) {
    return x->dtype == SIXI_SMP_BF16
               ? rope_dispatch<__nv_bfloat16, 8>(r, x, positions, n_tokens, head_dim, out, stream)
               : rope_dispatch<float, 4>(r, x, positions, n_tokens, head_dim, out, stream);
}

cudaError_t launch_kv_append(const KvGeom& g, const KvBatchView& b, const sixi_kv_tensor* k, const sixi_kv_tensor* v,
                             const RopeView& rope, uint32_t max_new, int32_t* status, uint32_t* seq_state,
                             cudaStream_t stream) {
    AppendArgs a;
    a.g = g, a.b = b, a.k = view_of(k), a.v = view_of(v), a.rope = rope, a.status = status, a.seq_state = seq_state;
    a.row_lanes = 2;
    while (a.row_lanes < g.head_dim / 8) a.row_lanes *= 2;
    const uint32_t rows = max_new < g.page_size ? max_new : g.page_size;
    // few rows: up to a warp a unit, so that many units share a CTA's way to them
    a.team = kNT;
    if (rows <= kRowsFew)
        for (a.team = a.row_lanes; a.team < 32u && a.team / a.row_lanes * kRowsHeld < rows;) a.team *= 2;
    const uint32_t teams = kNT / a.team;
    // A CTA's way to its rows is a chain of lookups, and the sines of a page's tokens are the same for every head. So with
    // a team of the whole CTA it takes up to four heads one after the other, while that leaves enough CTAs for the GPU.
    const uint32_t items = b.n_tokens / g.page_size + 2u * b.n_seqs;
    a.heads = 0;
    if (a.team == kNT) {
        a.heads = 4;
        while (a.heads > 1 && static_cast<uint64_t>(items) * 2u * ((g.n_heads + a.heads - 1) / a.heads) < 8u * 148u) a.heads /= 2;
    }
    const size_t table = rope.turns == nullptr ? 0 : static_cast<size_t>(g.page_size) * (rope.rot_dim / 2) * sizeof(float2);
    const int mode = table == 0 ? kAsIs : (a.heads > 1 && table <= kSinesMax ? kSharedSines : kOwnSines);
    const uint32_t units = a.heads ? 2u * ((g.n_heads + a.heads - 1) / a.heads) : (2u * g.n_heads + teams - 1) / teams;
    const dim3 grid(items, units);
    const size_t smem = mode == kSharedSines ? table : 0;
    const bool vec = view_aligned(k, g.n_heads, b.n_tokens) && view_aligned(v, g.n_heads, b.n_tokens) && rope_by_8(rope);
    const auto go = [&](auto kernel) {
        if (smem > 48u * 1024u) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (e != cudaSuccess) return e;
        }
        kernel<<<grid, kNT, smem, stream>>>(a);
        return cudaGetLastError();
    };
    const auto pick = [&](auto type) {
        using T = decltype(type);
        if (vec) {
            if (mode == kAsIs) return go(append_kernel<T, 8, kAsIs>);
            return mode == kSharedSines ? go(append_kernel<T, 8, kSharedSines>) : go(append_kernel<T, 8, kOwnSines>);
        }
        if (mode == kAsIs) return go(append_kernel<T, 1, kAsIs>);
        return mode == kSharedSines ? go(append_kernel<T, 1, kSharedSines>) : go(append_kernel<T, 1, kOwnSines>);
    };
    return k->dtype == SIXI_SMP_BF16 ? pick(__nv_bfloat16{}) : pick(float{});
}

cudaError_t launch_kv_read(const KvGeom& g, const KvBatchView& b, const sixi_kv_tensor* k, const sixi_kv_tensor* v,
                           int32_t* status, cudaStream_t stream) {
    ReadArgs a;
    a.g = g, a.b = b, a.k = view_of(k), a.v = view_of(v), a.status = status;
    // a token a warp while that does not fill the GPU (148 SMs of 8 such CTAs), up to four
    a.per = kNT / 32;
    while (a.per < 4 * (kNT / 32) && b.n_tokens / a.per > 148u * 16u) a.per *= 2;
    const uint32_t blocks = (b.n_tokens + a.per - 1) / a.per;
    const dim3 grid(blocks ? blocks : 1, 2);
    const bool vec = view_aligned(k, g.n_heads, b.n_tokens) && view_aligned(v, g.n_heads, b.n_tokens);
    if (k->dtype == SIXI_SMP_BF16) {
        if (vec) read_kernel<__nv_bfloat16, 8><<<grid, kNT, 0, stream>>>(a);
        else read_kernel<__nv_bfloat16, 1><<<grid, kNT, 0, stream>>>(a);
    } else {
        if (vec) read_kernel<float, 8><<<grid, kNT, 0, stream>>>(a);
        else read_kernel<float, 1><<<grid, kNT, 0, stream>>>(a);
    }
    return cudaGetLastError();
}

}  // namespace sixi_b200

// ---------------------------------------------------------------------------------------------
// extern "C"

using namespace sixi_b200;

struct sixi_kv {
    int32_t device;
    uint32_t n_sms;
    uint32_t max_seqs;
    KvGeom g;
    uint32_t* seq_state;  // [2 * max_seqs], zero between calls
    uint32_t* counter;    // [kAttnMaxCtas + 1], as AttnArgs has it
    float* part;          // attention's partial results
    CUtensorMap k_map, v_map;  // pages as attention copies them
};

struct sixi_kv_rope {
    int32_t device;
    RopeView v;
    uint64_t* d_turns;
};

namespace {

int32_t kv_from_cuda(cudaError_t e) {
    if (e == cudaSuccess) return SIXI_OK;
    if (e == cudaErrorMemoryAllocation) return SIXI_OUT_OF_MEMORY_VRAM;
    return SIXI_BACKEND_ERROR;
}

struct KvDeviceGuard {
    int prev = -1;
    explicit KvDeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) cudaSetDevice(dev);
    }
    ~KvDeviceGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

bool tensor_ok(const sixi_kv_tensor* t, uint64_t n_tokens) {
    if (t == nullptr || (t->dtype != SIXI_SMP_F32 && t->dtype != SIXI_SMP_BF16) || t->n_heads == 0) return false;
    if (n_tokens > 0 && t->data == nullptr) return false;
    return (reinterpret_cast<uintptr_t>(t->data) & (t->dtype == SIXI_SMP_BF16 ? 1u : 3u)) == 0;
}

// arrays that kernels read or write by elements of `size` bytes
bool aligned(const void* p, uintptr_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1u)) == 0; }

bool batch_ok(const sixi_kv* h, const sixi_kv_batch* b) {
    if (b == nullptr || b->n_seqs > h->max_seqs || b->n_tokens > 0x7FFFFFFFu) return false;
    if (b->n_seqs == 0) return b->n_tokens == 0;
    if (!aligned(b->offsets, 8) || !aligned(b->lens, 4) || !aligned(b->page_table, 4)) return false;
    // (positions of a tile's end and of a window's beginning stay within 31 bits)
    return b->offsets != nullptr && b->lens != nullptr && b->page_table != nullptr && b->table_stride >= b->max_pages &&
           b->max_pages > 0 && static_cast<uint64_t>(b->max_pages) * h->g.page_size <= (1ull << 30);
}

KvBatchView batch_view(const sixi_kv_batch* b) {
    return KvBatchView{b->page_table, b->table_stride, b->offsets, b->lens, b->n_seqs, b->max_pages, b->n_tokens};
}

// frequencies of a rotary configuration, in 64 bits
bool rope_frequencies(const sixi_kv_rope_config& c, std::vector<double>* inv, double* amp) {
    if (c.rot_dim < 2 || c.rot_dim > 256 || (c.rot_dim & 1u) || c.layout > SIXI_KV_ROPE_INTERLEAVED ||
        c.scaling > SIXI_KV_ROPE_YARN || !(c.base > 1.0) || !std::isfinite(c.base))
        return false;
    if (c.scaling != SIXI_KV_ROPE_NONE && (!(c.factor >= 1.0) || !std::isfinite(c.factor))) return false;
    const double d = c.rot_dim;
    const uint32_t n = c.rot_dim / 2;
    double base = c.base;
    if (c.scaling == SIXI_KV_ROPE_NTK) {
        if (c.rot_dim < 4) return false;
        base *= std::pow(c.factor, d / (d - 2.0));
    }
    inv->resize(n);
    for (uint32_t i = 0; i < n; ++i) (*inv)[i] = std::pow(base, -2.0 * i / d);
    *amp = 1.0;
    if (c.scaling == SIXI_KV_ROPE_LINEAR) {
        for (double& f : *inv) f /= c.factor;
    } else if (c.scaling == SIXI_KV_ROPE_YARN) {
        if (c.original_max_position < 1 || !(c.beta_slow > 0.0) || !(c.beta_fast >= c.beta_slow) ||
            !std::isfinite(c.beta_fast))
            return false;
        const double two_pi = 6.283185307179586476925;
        const auto at = [&](double turns) {
            return d * std::log(c.original_max_position / (turns * two_pi)) / (2.0 * std::log(c.base));
        };
        const double lo = std::fmax(0.0, std::floor(at(c.beta_fast)));
        const double hi = std::fmin(d - 1.0, std::ceil(at(c.beta_slow)));
        for (uint32_t i = 0; i < n; ++i) {
            const double r = std::fmin(1.0, std::fmax(0.0, (i - lo) / std::fmax(hi - lo, 1e-3)));
            (*inv)[i] = (*inv)[i] / c.factor * r + (*inv)[i] * (1.0 - r);
        }
        *amp = 0.1 * std::log(c.factor) + 1.0;
    }
    return true;
}

}  // namespace

extern "C" {

int32_t sixi_kv_create(int32_t device, const sixi_kv_config* c, void* k_pages, void* v_pages, float* k_scales,
                       float* v_scales, sixi_kv** out) {
    if (out == nullptr) return SIXI_INVALID_ARGUMENT;
    *out = nullptr;
    if (c == nullptr || k_pages == nullptr || v_pages == nullptr || k_scales == nullptr || v_scales == nullptr)
        return SIXI_INVALID_ARGUMENT;
    const uint32_t P = c->page_size;
    if ((P != 16 && P != 32 && P != 64 && P != 128) || c->n_pages == 0 || c->n_pages > 0x7FFFFFFFu || c->n_kv_heads == 0 ||
        c->n_kv_heads > 1024 || c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16 != 0 || c->max_seqs == 0 ||
        c->max_seqs > 65535)
        return SIXI_INVALID_ARGUMENT;
    // a tensor map's dimensions hold 32 bits
    if (static_cast<uint64_t>(c->n_pages) * c->n_kv_heads > 0x7FFFFFFFull) return SIXI_INVALID_ARGUMENT;
    if (((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15u) != 0 ||
        ((reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_scales)) & 3u) != 0)
        return SIXI_INVALID_ARGUMENT;
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n) return SIXI_INVALID_ARGUMENT;
    KvDeviceGuard guard(device);
    int major = 0, sms = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
        return SIXI_BACKEND_ERROR;
    if (major != 10) return SIXI_UNSUPPORTED_HARDWARE;
    sixi_kv* h = new (std::nothrow) sixi_kv;
    if (h == nullptr) return SIXI_BACKEND_ERROR;
    std::memset(h, 0, sizeof(*h));
    h->device = device;
    h->n_sms = static_cast<uint32_t>(sms);
    h->max_seqs = c->max_seqs;
    uint32_t shift = 0;
    while ((1u << shift) < P) ++shift;
    h->g = KvGeom{static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages), k_scales, v_scales, c->n_pages, P, shift,
                  c->n_kv_heads, c->head_dim};
    // 64 rows a CTA for one CTA per SM, or 16 for two
    const uint64_t part = 2ull * h->n_sms * part_floats(64, c->head_dim);
    cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&h->seq_state), sizeof(uint32_t) * 2u * c->max_seqs);
    if (e == cudaSuccess) e = cudaMalloc(reinterpret_cast<void**>(&h->counter), sizeof(uint32_t) * (kAttnMaxCtas + 1u));
    if (e == cudaSuccess)
        e = cudaMalloc(reinterpret_cast<void**>(&h->part), sizeof(float) * part);
    if (e == cudaSuccess) e = cudaMemset(h->seq_state, 0, sizeof(uint32_t) * 2u * c->max_seqs);
    if (e == cudaSuccess) e = cudaMemset(h->counter, 0, sizeof(uint32_t) * (kAttnMaxCtas + 1u));
    if (e == cudaSuccess) e = make_page_map(k_pages, h->g, &h->k_map);
    if (e == cudaSuccess) e = make_page_map(v_pages, h->g, &h->v_map);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {
        sixi_kv_destroy(h);
        return kv_from_cuda(e);
    }
    *out = h;
    return SIXI_OK;
}

int32_t sixi_kv_destroy(sixi_kv* h) {
    if (h == nullptr) return SIXI_OK;
    {
        KvDeviceGuard guard(h->device);
        if (h->seq_state) cudaFree(h->seq_state);
        if (h->counter) cudaFree(h->counter);
        if (h->part) cudaFree(h->part);
    }
    delete h;
    return SIXI_OK;
}

int32_t sixi_kv_rope_create(int32_t device, const sixi_kv_rope_config* c, sixi_kv_rope** out) {
    if (out == nullptr) return SIXI_INVALID_ARGUMENT;
    *out = nullptr;
    if (c == nullptr) return SIXI_INVALID_ARGUMENT;
    try {
        std::vector<double> inv;
        double amp = 1.0;
        if (!rope_frequencies(*c, &inv, &amp)) return SIXI_INVALID_ARGUMENT;
        int n = 0;
        if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n) return SIXI_INVALID_ARGUMENT;
        std::vector<uint64_t> turns(inv.size());
        for (size_t i = 0; i < inv.size(); ++i) {
            // f / (2 pi) < 1 turn per position; nearest 2^-64, held within 64 bits
            const long double t = static_cast<long double>(inv[i]) / 6.283185307179586476925286766559L;
            turns[i] = static_cast<uint64_t>(std::floor(std::ldexp(t, 64) + 0.5L));
        }
        KvDeviceGuard guard(device);
        sixi_kv_rope* r = new (std::nothrow) sixi_kv_rope;
        if (r == nullptr) return SIXI_BACKEND_ERROR;
        r->device = device;
        r->d_turns = nullptr;
        cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&r->d_turns), sizeof(uint64_t) * turns.size());
        if (e == cudaSuccess)
            e = cudaMemcpy(r->d_turns, turns.data(), sizeof(uint64_t) * turns.size(), cudaMemcpyHostToDevice);
        if (e != cudaSuccess) {
            sixi_kv_rope_destroy(r);
            return kv_from_cuda(e);
        }
        r->v = RopeView{r->d_turns, static_cast<float>(amp), static_cast<float>(amp), c->rot_dim,
                        c->layout == SIXI_KV_ROPE_INTERLEAVED ? 1u : 0u};
        *out = r;
        return SIXI_OK;
    } catch (...) {  // an allocation that failed: nothing passes the C boundary
        return SIXI_BACKEND_ERROR;
    }
}

int32_t sixi_kv_rope_destroy(sixi_kv_rope* r) {
    if (r == nullptr) return SIXI_OK;
    {
        KvDeviceGuard guard(r->device);
        if (r->d_turns) cudaFree(r->d_turns);
    }
    delete r;
    return SIXI_OK;
}

int32_t sixi_kv_rope_apply(const sixi_kv_rope* r, const sixi_kv_tensor* x, const int32_t* positions, uint32_t n_tokens,
                           uint32_t head_dim, uint32_t inverse, const sixi_kv_tensor* out, void* stream) {
    if (r == nullptr || !tensor_ok(x, n_tokens) || !tensor_ok(out, n_tokens) || x->dtype != out->dtype ||
        x->n_heads != out->n_heads || head_dim < r->v.rot_dim || head_dim > 65536)
        return SIXI_INVALID_ARGUMENT;
    if (n_tokens == 0) return SIXI_OK;
    if (positions == nullptr || !aligned(positions, 4) || n_tokens > 0x7FFFFFFFu) return SIXI_INVALID_ARGUMENT;
    KvDeviceGuard guard(r->device);
    RopeView view = r->v;
    if (inverse) view.amp_sin = -view.amp_sin;
    return kv_from_cuda(
        launch_rope_apply(view, x, positions, n_tokens, head_dim, out, static_cast<cudaStream_t>(stream)));
}

int32_t sixi_kv_append(sixi_kv* h, const sixi_kv_tensor* k, const sixi_kv_tensor* v, const sixi_kv_batch* b,
                       const sixi_kv_rope* rope, int32_t* out_status, void* stream) {
    if (h == nullptr || !batch_ok(h, b) || !tensor_ok(k, b->n_tokens) || !tensor_ok(v, b->n_tokens) ||
        k->dtype != v->dtype || k->n_heads != h->g.n_heads || v->n_heads != h->g.n_heads)
        return SIXI_INVALID_ARGUMENT;
    if (rope != nullptr && (rope->device != h->device || rope->v.rot_dim > h->g.head_dim)) return SIXI_INVALID_ARGUMENT;
    if (b->n_seqs == 0) return SIXI_OK;
    if (out_status == nullptr || !aligned(out_status, 4)) return SIXI_INVALID_ARGUMENT;
    KvDeviceGuard guard(h->device);
    const RopeView none{nullptr, 1.0f, 1.0f, 0u, 0u};
    return kv_from_cuda(launch_kv_append(h->g, batch_view(b), k, v, rope ? rope->v : none, b->max_new, out_status,
                                         h->seq_state, static_cast<cudaStream_t>(stream)));
}

int32_t sixi_kv_read(sixi_kv* h, const sixi_kv_batch* b, const sixi_kv_tensor* k, const sixi_kv_tensor* v,
                     int32_t* out_status, void* stream) {
    if (h == nullptr || !batch_ok(h, b) || !tensor_ok(k, b->n_tokens) || !tensor_ok(v, b->n_tokens) ||
        k->dtype != v->dtype || k->n_heads != h->g.n_heads || v->n_heads != h->g.n_heads)
        return SIXI_INVALID_ARGUMENT;
    if (b->n_seqs == 0) return SIXI_OK;
    if (out_status == nullptr || !aligned(out_status, 4)) return SIXI_INVALID_ARGUMENT;
    KvDeviceGuard guard(h->device);
    return kv_from_cuda(launch_kv_read(h->g, batch_view(b), k, v, out_status, static_cast<cudaStream_t>(stream)));
}

int32_t sixi_kv_attend(sixi_kv* h, const sixi_kv_tensor* q, const sixi_kv_batch* b, float scale, uint32_t window,
                       uint32_t flags, const sixi_kv_rope* rope, const sixi_kv_tensor* out, float* out_lse,
                       int32_t* out_status, void* stream) {
    if (h == nullptr || !batch_ok(h, b) || !tensor_ok(q, b->n_tokens) || !tensor_ok(out, b->n_tokens) ||
        q->dtype != out->dtype || q->n_heads != out->n_heads || q->n_heads % h->g.n_heads != 0 || !std::isfinite(scale) ||
        (flags & ~static_cast<uint32_t>(SIXI_KV_ATTEND_ALL)) != 0)
        return SIXI_INVALID_ARGUMENT;
    if (rope != nullptr && (rope->device != h->device || rope->v.rot_dim > h->g.head_dim)) return SIXI_INVALID_ARGUMENT;
    const uint64_t group = q->n_heads / h->g.n_heads;
    if (static_cast<uint64_t>(b->n_tokens) * group > 0x3FFFFFFFull) return SIXI_INVALID_ARGUMENT;
    if (b->n_seqs == 0) return SIXI_OK;
    // the schedule counts tiles (of 64 tokens and 8 rows at least) in 40 bits
    const double units = (b->n_tokens * static_cast<double>(group) / 8 + 2.0 * b->n_seqs) * h->g.n_heads;
    if (units * (b->max_pages * static_cast<double>(h->g.page_size) / 64 + 8) >= 1099511627776.0) return SIXI_INVALID_ARGUMENT;
    if (out_status == nullptr || !aligned(out_status, 4) || !aligned(out_lse, 4)) return SIXI_INVALID_ARGUMENT;
    KvDeviceGuard guard(h->device);
    AttnArgs a;
    std::memset(&a, 0, sizeof(a));
    a.g = h->g;
    a.b = batch_view(b);
    a.q = KvView{q->data, q->token_stride, q->head_stride};
    a.out = KvView{out->data, out->token_stride, out->head_stride};
    a.rope = rope ? rope->v : RopeView{nullptr, 1.0f, 1.0f, 0u, 0u};
    a.shape.group = static_cast<uint32_t>(group);
    a.shape.window = window >= 0x3FFFFFFFu ? 0u : window;  // wider than any sequence
    a.shape.all = (flags & SIXI_KV_ATTEND_ALL) ? 1u : 0u;
    a.shape.n_heads = h->g.n_heads;
    a.score = score_scale(scale);
    a.lse = out_lse;
    a.status = out_status;
    a.part = h->part;
    a.counter = h->counter;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return kv_from_cuda(q->dtype == SIXI_SMP_BF16
                            ? launch_attend_bf16(a, h->k_map, h->v_map, b->max_new, h->n_sms, s)
                            : launch_attend_f32(a, h->n_sms, s));
}

}  // extern "C"
