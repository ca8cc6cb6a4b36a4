// smp_kv.cuh - shared parts of the 8-bit paged key/value cache (include/sixi_kv.h): the handle, the
// device views of a call's arguments, e4m3 and rotary helpers, and the split of an attention call's
// work over a persistent grid.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "../../include/sixi_kv.h"

namespace sixi_b200 {

constexpr float kE4m3Max = 448.0f;
constexpr float kNegInf = -__builtin_huge_valf();

// ---------------------------------------------------------------------------------------------
// a call's arguments as the kernels see them

struct KvGeom {
    uint8_t* k_pages;
    uint8_t* v_pages;
    float* k_scales;
    float* v_scales;
    uint32_t n_pages, page_size, page_shift, n_heads, head_dim;
};

struct KvView {  // sixi_kv_tensor
    void* data;
    uint64_t token_stride, head_stride;
};

struct KvBatchView {
    const int32_t* page_table;
    uint64_t table_stride;
    const int64_t* offsets;
    const int32_t* lens;
    uint32_t n_seqs, max_pages, n_tokens;
};

struct RopeView {
    const uint64_t* turns;  // [rot_dim / 2] turns per position, as fractions of 2^64 (NULL: no rotation)
    float amp_cos, amp_sin;  // amp, and amp with the sign of the turn
    uint32_t rot_dim, interleaved;
};

// One sequence of a batch; n = 0 with ok = false when its numbers do not fit.
struct KvSeq {
    int64_t row0;  // first row in the call's tensors
    int32_t n, len;
    bool ok, in_order;  // in_order: its offsets are, and within the call's rows
};

__device__ __forceinline__ KvSeq kv_seq_of(const KvBatchView& b, uint32_t page_shift, int64_t r0, int64_t r1, int32_t len) {
    KvSeq q;
    q.row0 = r0;
    q.len = len;
    q.in_order = r0 >= 0 && r1 >= r0 && r1 <= static_cast<int64_t>(b.n_tokens);
    q.ok = q.in_order && len >= 0 &&
           static_cast<uint64_t>(len) <= (static_cast<uint64_t>(b.max_pages) << page_shift);
    q.n = q.ok ? static_cast<int32_t>(r1 - r0) : 0;
    return q;
}
__device__ __forceinline__ KvSeq kv_seq(const KvBatchView& b, uint32_t page_shift, uint32_t s) {
    return kv_seq_of(b, page_shift, b.offsets[s], b.offsets[s + 1], b.lens[s]);
}

// Whether the offsets from `at` on, `step` apart, are in order and within the call's rows. Where any is not, rows could
// belong to two sequences or to none, so every sequence of the call reports it.
__device__ __forceinline__ bool kv_offsets_ok(const KvBatchView& b, uint32_t at, uint32_t step) {
    bool ok = true;
    for (uint32_t s = at; s < b.n_seqs; s += step) {
        const int64_t r0 = b.offsets[s], r1 = b.offsets[s + 1];
        ok &= r0 >= 0 && r1 >= r0 && r1 <= static_cast<int64_t>(b.n_tokens);
    }
    return ok;
}

// ---------------------------------------------------------------------------------------------
// e4m3 and its power-of-two scales

// exponent e of the scale for a page whose largest magnitude is amax: the least e >= -126 with
// amax <= 448 * 2^e = 1.75 * 2^(e + 8); decided on the bits, so it is exact
__device__ __forceinline__ int kv_scale_exp(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;  // zero and subnormal amax: b >> 23 is 0
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
__device__ __forceinline__ int scale_exp_of(float s) { return static_cast<int>(__float_as_uint(s) >> 23) - 127; }

// two values to e4m3, nearest even, beyond 448 to 448
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t v) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xFFFFu), __NV_E4M3);
    return __half22float2(__half2(h));
}

// ---------------------------------------------------------------------------------------------
// from products to scores
//
// The factor is a significand times 2^(exponents of scale, query row, and page of keys). Queries and keys may have any
// magnitude that a float has, and theirs may cancel, so rows are brought to e4m3's range and the exponents are added as
// integers before anything is rounded.
struct ScoreScale {  // |scale| log2(e) = (1 + mant / 2^23) 2^exp; the sign (0: a scale of 0) goes to the queries
    uint32_t mant;
    int32_t exp;
    float sign;
};

inline ScoreScale score_scale(float scale) {
    int e = 0;
    float sig = static_cast<float>(2.0 * std::frexp(std::fabs(static_cast<double>(scale)) * 1.4426950408889634, &e));
    if (sig >= 2.0f) sig = 1.0f, ++e;  // (it was in [1, 2) before it was rounded)
    ScoreScale s;
    std::memcpy(&s.mant, &sig, sizeof(sig));
    s.mant &= 0x7FFFFFu;
    s.exp = e - 1;
    s.sign = scale < 0.0f ? -1.0f : (scale > 0.0f ? 1.0f : 0.0f);
    return s;
}

// A row's code, its elements divided by 2^e: its exponents in bits 23 up (plus 256), the significand below. Beyond what a
// float holds the factor ends at 2^-126 (products are below 2^26, so scores are nothing there) or at 2^127.
__device__ __forceinline__ uint32_t score_code(const ScoreScale& s, int e) {
    return static_cast<uint32_t>(min(max(e + s.exp, -256), 255) + 256) << 23 | s.mant;
}
__device__ __forceinline__ float score_factor(uint32_t code, int ek) {
    const int e = min(max(static_cast<int>(code >> 23) - 256 + ek, -126), 127);
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23 | (code & 0x7FFFFFu));
}

// ---------------------------------------------------------------------------------------------
// element access: VEC consecutive elements as fp32 (VEC = 1, or 8 with 16-byte alignment)

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
    if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 4) x[0] = *reinterpret_cast<const float*>(p);
        else x[0] = __bfloat162float(*p);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + i);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i + 2 * j] = __uint_as_float(w[j] << 16);
                x[i + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            }
        }
    }
}

__device__ __forceinline__ uint32_t bf16x2_bits(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
    if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float*>(p) = x[0];
        else *p = __float2bfloat16_rn(x[0]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4)
            *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 8) {
            uint4 v;
            v.x = bf16x2_bits(x[i], x[i + 1]), v.y = bf16x2_bits(x[i + 2], x[i + 3]);
            v.z = bf16x2_bits(x[i + 4], x[i + 5]), v.w = bf16x2_bits(x[i + 6], x[i + 7]);
            *reinterpret_cast<uint4*>(p + i) = v;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// rotary positions

// sin and cos of position * f for a frequency held as a 64-bit fraction of a turn: the product wraps
// at whole turns, so only the angle within a turn is ever rounded (to 2^-32 of a turn, then to fp32).
__device__ __forceinline__ void rope_sincos(const RopeView& r, int32_t pos, uint32_t pair, float* s, float* c) {
    const uint64_t frac = static_cast<uint64_t>(static_cast<int64_t>(pos)) * r.turns[pair];
    const int32_t half_turns = static_cast<int32_t>(static_cast<uint32_t>((frac + 0x80000000ull) >> 32));
    sincospif(static_cast<float>(half_turns) * 4.656612873077393e-10f /* 2^-31 */, s, c);
    *s *= r.amp_sin;
    *c *= r.amp_cos;
}

// Elements [i0, i0 + VEC) of the head at p, turned by pos (fp32). VEC consecutive elements are all
// turned or all passed through, and in the half layout lie in one half (VEC divides rot_dim / 2 then,
// and rot_dim in the interleaved one).
template <typename T, int VEC>
__device__ __forceinline__ void load_turned(const RopeView& r, const T* p, uint32_t i0, int32_t pos, float* x) {
    load_vec<T, VEC>(p + i0, x);
    if (r.turns == nullptr || i0 >= r.rot_dim) return;
    float s, c;
    if (r.interleaved) {
        if constexpr (VEC == 1) {
            float o;
            load_vec<T, 1>(p + (i0 ^ 1u), &o);
            rope_sincos(r, pos, i0 >> 1, &s, &c);
            x[0] = (i0 & 1u) ? x[0] * c + o * s : x[0] * c - o * s;
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                rope_sincos(r, pos, (i0 + j) >> 1, &s, &c);
                const float a = x[j], b = x[j + 1];
                x[j] = a * c - b * s;
                x[j + 1] = b * c + a * s;
            }
        }
    } else {
        const uint32_t half = r.rot_dim >> 1;
        const bool upper = i0 >= half;
        float o[VEC];
        load_vec<T, VEC>(p + (upper ? i0 - half : i0 + half), o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            rope_sincos(r, pos, (upper ? i0 - half : i0) + j, &s, &c);
            x[j] = upper ? x[j] * c + o[j] * s : x[j] * c - o[j] * s;
        }
    }
}

__device__ __forceinline__ void unpack8(uint4 v, float* x) {  // 8 bf16
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
}

// ---------------------------------------------------------------------------------------------
// attention: how a call's work is cut

// The rows of a (sequence, key head) are its new tokens times the G query heads of the key head,
// row r = token * G + g. A unit is a row tile of `rt` rows; it reads the tokens of tiles [first, end)
// of `T` tokens. Units are laid out on one line of (virtual) tiles, sequence by sequence, head by
// head, and CTA c of n takes [total * c / n, total * (c + 1) / n): every CTA gets the same number of
// tiles whatever the lengths are, and a unit may span several CTAs, whose partial results the last
// one to arrive joins in CTA order. With many row tiles of a causal prompt, tile j is laid next to
// tile nr - 1 - j: the pair's length hardly varies, so that the line needs no prefix sum over row
// tiles. A pair (or a lone unit) takes `weight` virtual tiles; what its units leave is idle.
struct AttnShape {
    uint32_t group, rt, tile_shift, window, all, n_heads;
    // Beginning and ending a unit takes about as long as this many of its tiles: each unit's place on the line is so much
    // longer than its tiles, and CTAs with many short units get fewer tiles.
    uint32_t unit_cost;
    uint32_t whole_tiles;  // units of at most this many tiles (in every sequence of a call) are not cut
};

// 64-bit quotient; the 32-bit one, which is much shorter, where it is enough
__device__ __forceinline__ uint64_t quot(uint64_t a, uint64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

struct SeqPlan {
    int32_t n, len;       // new tokens, length
    int64_t row0;
    int32_t p0;           // position of the first new token (negative: empty rows)
    uint32_t nr;          // row tiles
    uint32_t paired;      // row tiles laid in pairs
    uint32_t weight;      // virtual tiles of a pair or unit
    uint32_t lanes;       // pairs or units per head
    bool in_order;        // as KvSeq
};

__device__ __forceinline__ void unit_tiles(const AttnShape& a, const SeqPlan& s, uint32_t j, int32_t* first,
                                           int32_t* end) {
    const uint32_t r0 = j * a.rt;
    const uint32_t last = min(r0 + a.rt, static_cast<uint32_t>(s.n) * a.group) - 1u;
    const int32_t hi = a.all ? s.len - 1 : min(s.len - 1, s.p0 + static_cast<int32_t>(last / a.group));
    int32_t lo = 0;
    if (a.window) lo = max(0, s.p0 + static_cast<int32_t>(r0 / a.group) - static_cast<int32_t>(a.window) + 1);
    lo = min(lo, max(hi, 0));
    *first = lo >> a.tile_shift;
    *end = (max(hi, 0) >> a.tile_shift) + 1;  // a unit without positions still takes one (empty) tile
}

__device__ __forceinline__ SeqPlan plan_seq(const AttnShape& a, const KvBatchView& b, uint32_t page_shift, uint32_t s) {
    const KvSeq q = kv_seq(b, page_shift, s);
    SeqPlan p;
    p.n = q.n, p.len = q.ok ? q.len : 0, p.row0 = q.row0, p.in_order = q.in_order;
    p.p0 = p.len - p.n;
    const uint32_t rows = static_cast<uint32_t>(p.n) * a.group;
    p.nr = (rows + a.rt - 1) / a.rt;
    p.paired = 0;
    p.weight = 0;
    p.lanes = p.nr;
    if (p.nr == 0) return p;
    int32_t f0, e0, f1, e1;
    unit_tiles(a, p, p.nr - 1, &f1, &e1);
    if (p.nr == 1) {
        p.weight = static_cast<uint32_t>(e1 - f1) + a.unit_cost;
        return p;
    }
    // bound of one unit: the last row tile's, and under a window what the window and the tile's own
    // positions can span
    const uint32_t span = (a.rt - 1) / a.group + 2;
    uint32_t one = static_cast<uint32_t>(e1);
    if (a.window && !a.all) one = min(one, ((a.window + span) >> a.tile_shift) + 2u);
    unit_tiles(a, p, 0, &f0, &e0);
    // bound of a pair: floor(x / T) + floor(y / T) <= floor((x + y) / T) for the two last positions
    const uint64_t reach = 2ull * static_cast<uint64_t>(max(p.p0, 0)) +
                           quot(static_cast<uint64_t>(p.nr + 1) * a.rt, a.group);
    const uint32_t two = min(static_cast<uint32_t>((reach >> a.tile_shift) + 2u), 2u * one);
    const uint64_t flat = static_cast<uint64_t>(p.nr) * (one + a.unit_cost);
    const uint64_t pair = static_cast<uint64_t>((p.nr + 1) / 2) * (two + 2u * a.unit_cost);
    p.paired = (pair < flat && !a.all) ? 1u : 0u;
    p.weight = p.paired ? two + 2u * a.unit_cost : one + a.unit_cost;
    p.lanes = p.paired ? (p.nr + 1) / 2 : p.nr;
    return p;
}

__device__ __forceinline__ uint64_t plan_tiles(const AttnShape& a, const SeqPlan& p) {
    return static_cast<uint64_t>(p.weight) * p.lanes * a.n_heads;
}

// A piece of a unit that one CTA works on: token tiles [t0, t1) of the unit's [first, end).
struct Piece {
    uint32_t seq, head, row_tile, rows;  // rows: valid rows of the row tile
    int32_t t0, t1, first, end;
    uint64_t start;  // the unit's place on the line
    SeqPlan plan;
};

// Walks the pieces of one CTA's range. All threads of a role walk it alike.
struct PieceWalk {
    uint64_t at, stop;       // this CTA's range, `at` moving on
    uint64_t seq_at;         // where the current sequence starts
    uint32_t seq;
    SeqPlan plan;
    bool loaded;
    bool whole;  // the line is one of units, not tiles: no unit is cut
};

__device__ __forceinline__ bool next_piece(const AttnShape& a, const KvBatchView& b, uint32_t page_shift, PieceWalk& w,
                                           Piece* out) {
    while (w.at < w.stop) {
        if (!w.loaded) {
            if (w.seq >= b.n_seqs) return false;
            w.plan = plan_seq(a, b, page_shift, w.seq);
            w.loaded = true;
        }
        const uint64_t all = w.whole ? static_cast<uint64_t>(w.plan.lanes) * a.n_heads : plan_tiles(a, w.plan);
        if (w.at >= w.seq_at + all) {
            w.seq_at += all;
            ++w.seq;
            w.loaded = false;
            continue;
        }
        const uint64_t in_seq = w.at - w.seq_at;
        const uint64_t lane = w.whole ? in_seq : quot(in_seq, w.plan.weight);
        const uint32_t head = static_cast<uint32_t>(quot(lane, w.plan.lanes));
        const uint32_t slot = static_cast<uint32_t>(lane - static_cast<uint64_t>(head) * w.plan.lanes);
        uint32_t off = w.whole ? 0u : static_cast<uint32_t>(in_seq - lane * w.plan.weight);
        uint64_t start = w.whole ? w.at : w.seq_at + lane * w.plan.weight;
        uint32_t j = slot;
        int32_t first, end;
        unit_tiles(a, w.plan, j, &first, &end);
        if (off >= static_cast<uint32_t>(end - first)) {
            const uint32_t mate = w.plan.nr - 1 - slot;
            const uint32_t used = static_cast<uint32_t>(end - first);
            if (w.plan.paired && mate != slot) {
                start += used;
                off -= used;
                j = mate;
                unit_tiles(a, w.plan, j, &first, &end);
            }
            if (off >= static_cast<uint32_t>(end - first)) {  // idle rest of the pair's place
                w.at = w.seq_at + (lane + 1) * w.plan.weight;
                continue;
            }
        }
        const uint64_t left = w.whole ? ~0ull : w.stop - w.at;
        const uint32_t have = static_cast<uint32_t>(end - first) - off;
        const uint32_t take = left < have ? static_cast<uint32_t>(left) : have;
        out->seq = w.seq;
        out->head = head;
        out->row_tile = j;
        out->rows = min(a.rt, static_cast<uint32_t>(w.plan.n) * a.group - j * a.rt);
        out->first = first;
        out->end = end;
        out->t0 = first + static_cast<int32_t>(off);
        out->t1 = out->t0 + static_cast<int32_t>(take);
        out->start = start;
        out->plan = w.plan;
        w.at += w.whole ? 1u : take;
        return true;
    }
    return false;
}

// The line's total and this CTA's start on it: every thread of the block calls (NT threads); `scratch` is NT / 32 + 2
// shared 64-bit words, `found` takes the plan of the sequence that the CTA starts in, `disorder` (shared, zero before)
// whether any sequence's offsets are out of order. Returns false when the CTA has nothing to do. *ctas: CTAs that share the
// line.
template <int NT>
__device__ __forceinline__ bool walk_init(const AttnShape& a, const KvBatchView& b, uint32_t page_shift,
                                          unsigned long long* scratch, SeqPlan* found, uint32_t* disorder, PieceWalk* w,
                                          uint64_t* total_out, uint32_t* ctas) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr uint64_t kTiles = (1ull << 40) - 1ull;  // tiles in the low 40 bits, units above them
    uint64_t total = 0;
    uint32_t n = 0;
    bool whole = true;
    const bool one_chunk = b.n_seqs <= NT;
    for (uint32_t pass = 0; pass < 2; ++pass) {
        uint64_t before = 0;
        for (uint32_t s0 = 0; s0 < b.n_seqs; s0 += NT) {
            const uint32_t s = s0 + threadIdx.x;
            uint64_t mine = 0;
            SeqPlan p;
            bool small = true, in_order = true;
            if (s < b.n_seqs) {
                p = plan_seq(a, b, page_shift, s);
                mine = plan_tiles(a, p) | (static_cast<uint64_t>(p.lanes) * a.n_heads << 40);
                small = !p.paired && p.weight <= a.whole_tiles + a.unit_cost;
                in_order = p.in_order;
            }
            uint64_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t t = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= o) incl += t;
            }
            __syncthreads();
            if (lane == 31) scratch[warp] = incl;
            if (!in_order) *disorder = 1u;
            if (pass == 0) whole = __syncthreads_and(small && whole) != 0;
            else __syncthreads();
            uint64_t all = 0, prev = 0;
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) {
                const uint64_t t = scratch[i];
                prev += i < warp ? t : 0;
                all += t;
            }
            if (pass == 0) total += all;
            if (pass == 1 || one_chunk) {
                if (s0 == 0) {
                    // (beyond 2^20 tiles the unit count may not hold its bits, and no unit is small enough to matter)
                    whole = whole && (total & kTiles) < (1u << 20);
                    total = whole ? total >> 40 : total & kTiles;
                    n = total < gridDim.x ? static_cast<uint32_t>(total) : gridDim.x;
                }
                if (blockIdx.x < n) {
                    const uint64_t at = quot(total * blockIdx.x, n);
                    const uint64_t lo64 = before + prev + incl - mine;
                    const uint64_t lo = whole ? lo64 >> 40 : lo64 & kTiles, len = whole ? mine >> 40 : mine & kTiles;
                    if (at >= lo && at < lo + len) {
                        scratch[NT / 32] = s;
                        scratch[NT / 32 + 1] = lo;
                        *found = p;
                    }
                }
            }
            before += all;
        }
        if (one_chunk) break;  // one round has both
    }
    __syncthreads();
    *total_out = total;
    *ctas = n;
    if (blockIdx.x >= n) return false;
    w->at = quot(total * blockIdx.x, n);
    w->stop = quot(total * (blockIdx.x + 1), n);
    w->seq = static_cast<uint32_t>(scratch[NT / 32]);
    w->seq_at = scratch[NT / 32 + 1];
    w->plan = *found;
    w->loaded = true;
    w->whole = whole;
    return true;
}

// whether a sequence's numbers and the page ids that its rows need are in range (a warp or block
// strides over the ids: `at` of `step` threads)
__device__ __forceinline__ bool seq_pages_ok(const AttnShape& a, const KvBatchView& b, uint32_t page_shift,
                                             uint32_t n_pages, uint32_t s, uint32_t at, uint32_t step) {
    const KvSeq q = kv_seq(b, page_shift, s);
    bool ok = q.ok;
    if (q.n > 0 && q.len > 0) {
        int32_t lo = 0;
        if (a.window) lo = max(0, q.len - q.n - static_cast<int32_t>(a.window) + 1);
        const uint32_t p1 = static_cast<uint32_t>(q.len - 1) >> page_shift;
        for (uint32_t p = (static_cast<uint32_t>(lo) >> page_shift) + at; p <= p1; p += step)
            ok &= static_cast<uint32_t>(b.page_table[s * b.table_stride + p]) < n_pages;
    }
    return ok;
}

// CTA that owns place x when n CTAs share `total` places (n <= total)
__device__ __forceinline__ uint32_t place_owner(uint64_t x, uint64_t total, uint32_t n) {
    return static_cast<uint32_t>(quot((x + 1) * n - 1, total));
}

// ---------------------------------------------------------------------------------------------
// launches (host)

constexpr uint32_t kAttnMaxCtas = 512;  // CTAs of an attention call at most

struct AttnArgs {
    KvGeom g;
    KvBatchView b;
    KvView q, out;
    RopeView rope;
    AttnShape shape;
    ScoreScale score;
    float* lse;
    int32_t* status;
    float* part;        // [2 * ctas][part_stride]
    uint32_t* counter;  // [kAttnMaxCtas], zero between calls; then one word: a wait of a call has run out
    uint64_t part_stride;
};

// whether 8 consecutive elements (at a multiple of 8) are turned, or passed through, together
inline bool rope_by_8(const RopeView& r) {
    return r.turns == nullptr || (r.interleaved ? r.rot_dim % 8 == 0 : (r.rot_dim / 2) % 8 == 0);
}

// Partial results: two per CTA (a unit that the CTA continues, and one that it leaves to the next), each the row tile's
// rows of head_dim unnormalised fp32 sums, then the rows' maxima (base 2) and sums. They lie close together: a step over
// a large cache keeps few address translations alive, and joining results that were megabytes apart took 10 us more.
inline uint64_t part_floats(uint32_t rows, uint32_t head_dim) { return static_cast<uint64_t>(rows) * (head_dim + 2u); }

// ---------------------------------------------------------------------------------------------
// joining the pieces of a unit

__device__ __forceinline__ float kv_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Eight warps (w: 0 to 7) join a unit's n pieces in CTA order: piece 0 is its CTA's last result (first), the others are
// their CTAs' first ones (rest + 2 c results on). Rows of `rt`-row results; row r goes to query token
// (row_base + r) / group of row0 on. DC: 128-element chunks of a head; U rows at a time, the loads of kAhead pieces in
// flight: a round is a chain of loads, so units of many rows (and then few pieces) take more rows at a time.
template <typename T, int DC, int U, int kAhead>
__device__ __forceinline__ void join_rows(const AttnArgs& a, const float* first, const float* rest, uint32_t n, uint32_t rows,
                                          uint32_t row_base, int64_t row0, uint32_t head, uint32_t w) {
    const uint32_t lane = threadIdx.x & 31u, D = a.g.head_dim;
    const auto piece_of = [&](uint32_t c) { return c == 0 ? first : rest + 2ull * c * a.part_stride; };
    // a warp a row, four elements a lane, U rows at a time; a lane holds the factor of a piece (of every 32nd)
    for (uint32_t r0 = w; r0 < rows; r0 += 8u * U) {
        uint32_t row[U];
        float m[U], l[U], f[U], norm[U];
        float4 o[U][DC], v[U][DC][kAhead];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            row[u] = min(r0 + 8u * u, rows - 1u);
            m[u] = kNegInf, l[u] = 0.0f;
#pragma unroll
            for (int k = 0; k < DC; ++k) o[u][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        // (the first pieces' sums are on their way before the factors are known)
        const auto fetch = [&](uint32_t c) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < DC; ++k)
#pragma unroll
                    for (int i = 0; i < kAhead; ++i)
                        if (k * 128u + lane * 4u < D)
                            v[u][k][i] = __ldcg(reinterpret_cast<const float4*>(piece_of(min(c + i, n - 1u)) + row[u] * D +
                                                                                k * 128u + lane * 4u));
        };
        fetch(0);
        for (uint32_t c = lane; c < n; c += 32u)
#pragma unroll
            for (int u = 0; u < U; ++u) m[u] = fmaxf(m[u], __ldcg(piece_of(c) + a.shape.rt * D + row[u]));
#pragma unroll
        for (int o2 = 16; o2 > 0; o2 >>= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) m[u] = fmaxf(m[u], __shfl_xor_sync(0xFFFFFFFFu, m[u], o2));
        for (uint32_t c0l = 0; c0l < n; c0l += 32u) {
            const uint32_t c = c0l + lane;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                f[u] = 0.0f;
                if (c < n) {
                    const float* p = piece_of(c) + a.shape.rt * D + row[u];
                    const float mc = __ldcg(p);
                    f[u] = mc == m[u] ? 1.0f : kv_ex2(mc - m[u]);
                    l[u] += __ldcg(p + a.shape.rt) * f[u];
                }
            }
            for (uint32_t i0 = 0; i0 < 32u && c0l + i0 < n; i0 += kAhead) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const float g = __shfl_sync(0xFFFFFFFFu, f[u], i0 + i);  // (0 past the last piece)
#pragma unroll
                        for (int k = 0; k < DC; ++k) {
                            if (g == 0.0f) continue;
                            o[u][k].x = fmaf(v[u][k][i].x, g, o[u][k].x), o[u][k].y = fmaf(v[u][k][i].y, g, o[u][k].y);
                            o[u][k].z = fmaf(v[u][k][i].z, g, o[u][k].z), o[u][k].w = fmaf(v[u][k][i].w, g, o[u][k].w);
                        }
                    }
                if (c0l + i0 + kAhead < n) fetch(c0l + i0 + kAhead);
            }
        }
#pragma unroll
        for (int o2 = 16; o2 > 0; o2 >>= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) l[u] += __shfl_xor_sync(0xFFFFFFFFu, l[u], o2);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r0 + 8u * u >= rows) continue;
            norm[u] = l[u] == 0.0f ? 0.0f : 1.0f / l[u];
            const uint32_t rr = row_base + row[u], tok = rr / a.shape.group;
            const uint32_t hq = head * a.shape.group + rr - tok * a.shape.group;
            if (a.lse && lane == 0)
                a.lse[(row0 + tok) * (a.shape.n_heads * a.shape.group) + hq] = (m[u] + log2f(l[u])) * 0.6931471805599453f;
            T* p = static_cast<T*>(a.out.data) + (row0 + tok) * a.out.token_stride + hq * a.out.head_stride;
#pragma unroll
            for (int k = 0; k < DC; ++k)
                if (k * 128u + lane * 4u < D) {
                    const float y[4] = {o[u][k].x * norm[u], o[u][k].y * norm[u], o[u][k].z * norm[u], o[u][k].w * norm[u]};
#pragma unroll
                    for (int i = 0; i < 4; ++i) store_vec<T, 1>(p + k * 128u + lane * 4u + i, y + i);
                }
        }
    }
}

cudaError_t launch_rope_apply(const RopeView& r, const sixi_kv_tensor* x, const int32_t* positions, uint32_t n_tokens,
                              uint32_t head_dim, const sixi_kv_tensor* out, cudaStream_t stream);
cudaError_t launch_kv_append(const KvGeom& g, const KvBatchView& b, const sixi_kv_tensor* k, const sixi_kv_tensor* v,
                             const RopeView& rope, uint32_t max_new, int32_t* status, uint32_t* seq_state,
                             cudaStream_t stream);
cudaError_t launch_kv_read(const KvGeom& g, const KvBatchView& b, const sixi_kv_tensor* k, const sixi_kv_tensor* v,
                           int32_t* status, cudaStream_t stream);
cudaError_t launch_attend_f32(AttnArgs a, uint32_t n_sms, cudaStream_t stream);
cudaError_t make_page_map(void* pages, const KvGeom& g, CUtensorMap* out);
cudaError_t launch_attend_bf16(const AttnArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map, uint32_t max_new,
                               uint32_t n_sms, cudaStream_t stream);

}  // namespace sixi_b200
