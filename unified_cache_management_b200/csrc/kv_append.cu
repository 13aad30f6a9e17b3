// Append of a step's keys and values to the paged KV cache (sm_100a), the keys rotated on the way; in the same launch the
// step's queries are rotated, and the rotated keys are also written out in 16 bits for callers that hash them.
//
// Cache of 16-bit values: rows are stored as they are (keys: rotated in float32, rounded once).
// Cache of e4m3 codes with one float32 scale per (block, kv head): value = code * scale, scale = the smallest power of two
// with 448 * scale >= the block's largest finite value (448 = largest e4m3).  A power of two costs no precision (e4m3 is
// a float format: only values below 2^-15 of the largest lose bits), and when a block's scale has to grow, the codes
// that are there already move by an exponent - exact, but for codes that become subnormal.
//   - a call that writes row 0 of a block starts the block anew: the scale comes from this call's rows alone, other rows
//     keep their codes and lose their meaning;
//   - otherwise the block keeps max(old scale, scale needed by the new rows); if that grows, the codes of all rows that
//     this call does not write are re-rounded to the new scale;
//   - a value that is not finite is stored as NaN (e4m3 has no infinity) and has no say in the scale; the scale of a block
//     whose values are all zero is 0.
//
// One owner per block: since a block's scale depends on all of its new rows, and its old rows may have to be rewritten,
// one CTA (per head group) handles all rows of a block that the call touches.  A CTA looks at `chunk` consecutive tokens;
// each that begins a run of tokens of one block is a candidate, and the CTA walks the whole slot list once for other
// tokens of its candidates' blocks (a 1024-bit filter in front).  The candidate with the block's first token owns it; if
// a slot is listed twice, the later token's row is the one that is stored.  So the result does not depend on the order
// in which CTAs run, whatever the order of the slot list, and no atomic touches global memory.
// The walk costs T / chunk * head groups * T slot reads out of L2: 67 MB for 32768 tokens in blocks and chunks of 128 with
// one head group, next to 740 MB of HBM traffic that such a call (8 + 32 heads of 128, e4m3) cannot do without.  It grows with the
// square of T, so a call takes kAppMaxTokens tokens at most (a terabyte of L2 reads).
//
// Keys and values of a candidate go to the two halves of the CTA (256 threads each), in turn, since keys take longer.  A half
// goes over the rows of one head of the block twice, first for the largest value, then, out of L2, for the codes.  Cosines
// and sines of a tile of rows are computed once per block, in shared memory, for all heads.  HBM-bound in principle (2 bytes
// read and 1 written per element); what it does reach is set by latency and instruction issue: two CTAs of 512 threads fit an
// SM with 64 registers a thread.  Measured for the call above: 180 us, 84 us of it the queries' rotation (at its floor);
// keys and values alone 92 us, 67 us without rotation, where their bytes would take 31 us; four times the tokens 448 us, sixteen
// times 3570 us, by the walk.  The rotated keys written out besides: 208 us.  Tried and slower: values held in registers between the passes (234 us in all), halves of 128 threads, one or three CTAs per SM.
// A decode step of 16 tokens takes 7.4 us in a graph (6.0 us for 16-bit caches), bound by latency: walk, filter, rows, two passes.
#include <cuda_fp8.h>

#include "rotary.cuh"

namespace ucmr {

int device_sms();

constexpr int kAppHalf = 256;              // threads per half
constexpr int kAppTile = 16384;            // elements of a head whose cosines and sines are in shared memory: 64 KB
constexpr int kAppMaxChunk = 128;
constexpr int kAppMaxBlock = 1024;         // rows per block
constexpr int kAppMaxTokens = 1 << 22;     // per call
constexpr int kAppList = 1024;             // (candidate, token) pairs that the walk may find before it is repeated per candidate

struct AppendJob {
    const void* x[2];       // keys, values [T, Hkv, D]
    int64_t xs_t[2], xs_h[2];
    void* cache[2];         // [NB, BS, Hkv, D]
    int64_t cs_b[2], cs_t[2], cs_h[2];
    float* scale[2];        // [NB, Hkv] or null
    const void* slots;
    int slot_is_int64;
    int64_t T, NB;
    int BS, Hkv, D;
    int chunk, heads_per_cta, head_tiles;
    FastDiv by_row, by_block;   // divisions by the items of a row, D / 16, and by BS
};

struct AppendParams {
    RotaryAngles ang;       // inv_freq null: keys are stored as they come
    AppendJob store;
    RotaryJob rot[2];       // queries, copy of the rotated keys (T = 0: none)
    int64_t rot_ctas[2];
    int rot_vector[2];
};

__device__ __forceinline__ void half_sync(int half) { asm volatile("bar.sync %0, %1;" ::"r"(half + 1), "n"(kAppHalf) : "memory"); }

// Sixteen elements of a row -> float32.  Keys with a rotation: item `ch` < rot/16 holds eight pairs; the others and all
// values are 16 consecutive elements.
struct ItemPlace { int first, second; };

__device__ __forceinline__ ItemPlace item_place(bool rotated, const RotaryAngles& ang, int ch)
{
    ItemPlace p;
    if (rotated && ch < ang.rot / 16) pair_offsets(ang.rot, ang.interleaved, ch, p.first, p.second);
    else { p.first = ch * 16; p.second = p.first + 8; }
    return p;
}

template <typename T>
__device__ __forceinline__ void item_values(uint4 va, uint4 vb, bool turn, const float4* cs, int step, int interleaved,
                                            float (&a)[8], float (&b)[8])
{
    if (turn) {
        rotate_pairs<T>(va, vb, cs, step, interleaved, a, b);
        return;
    }
    const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 fa = Half2<T>::to_float(wa[i]), fb = Half2<T>::to_float(wb[i]);
        a[2 * i] = fa.x; a[2 * i + 1] = fa.y;
        b[2 * i] = fb.x; b[2 * i + 1] = fb.y;
    }
}

// Exponent e of the scale 2^e for a largest value `m` > 0: 448 = 1.75 * 2^8.  Kept at -126 or more, so that the scale and
// its reciprocal are normal numbers.
__device__ __forceinline__ float scale_for(float m)
{
    if (!(m > 0.f)) return 0.f;
    const uint32_t bits = __float_as_uint(m);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, -126);  // (a subnormal m lands here too)
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Reciprocal of a scale: exact for a power of two.  A scale that a caller brought may be anything else; kept finite, so that
// zeros stay zeros.
__device__ __forceinline__ float inverse_scale(float s) { return s > 0.f ? fminf(1.0f / s, 3.402823466e38f) : 0.f; }

// Four codes, rounded to nearest, |values| up to 448 or NaN.  ODD: values may be infinite, which the saturating conversion
// would make 448: they become NaN.
template <bool ODD>
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d)
{
    if (ODD) {
        const float inf = __uint_as_float(0x7f800000u), nan = __uint_as_float(0x7fffffffu);
        a = fabsf(a) == inf ? nan : a; b = fabsf(b) == inf ? nan : b;
        c = fabsf(c) == inf ? nan : c; d = fabsf(d) == inf ? nan : d;
    }
    uint16_t lo, hi;  // (the second operand goes to the low byte)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

__device__ __forceinline__ void from_e4m3x4(uint32_t w, float (&f)[4])
{
    uint32_t lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
    const float2 a = __half22float2(reinterpret_cast<const __half2&>(lo)), b = __half22float2(reinterpret_cast<const __half2&>(hi));
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}

template <bool ODD>
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inv)
{
    return make_uint2(to_e4m3x4<ODD>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                      to_e4m3x4<ODD>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}

// Shared memory of the store: cosines and sines of a tile's rows (rows * rot/16 * 64 bytes), then the control words.
struct AppendCtl {
    int64_t cand_block[kAppMaxChunk];
    int cand_token[kAppMaxChunk];
    int lead[kAppMaxChunk];
    uint32_t filter[32];
    int list_cand[kAppList];
    int list_token[kAppList];
    int n_cand, n_list, n_rows;
    int row_token[kAppMaxBlock];   // token of each row of the block in hand, -1 = not written
    int rows[kAppMaxBlock];        // the rows that are written
    int tokens[kAppMaxBlock];      // and their tokens
    uint32_t big[2][4];            // largest value of a half's rows, as bits, and largest finite one; heads take them in turn
    int warp_count[kAppMaxChunk / 32];
};

__device__ __forceinline__ uint32_t filter_bit(int64_t block) { return ((uint32_t)block * 2654435761u) >> 22; }

// Cosines and sines of the rows [r0, r0 + nr) of the block in hand, by `threads` threads.
__device__ __forceinline__ void fill_tile(const AppendParams& p, float4* cs, const AppendCtl* ctl, int r0, int nr, int tid, int threads)
{
    const int np = p.ang.rot / 2, chunks = p.ang.rot / 16;
    for (int i = tid; i < nr * np; i += threads) {
        const int row = i / np;
        fill_cos_sin(cs, p.ang, load_index(p.ang.positions, p.ang.pos_is_int64, ctl->tokens[r0 + row]), row, i - row * np, chunks);
    }
}

// One half of the CTA stores the keys (kind 0) or the values (kind 1) of one head of the block in hand.  `turn`: which of the
// half's heads this is.  The cosines of a block that is one tile are there already.
template <typename T, bool CODES, bool TURN>
__device__ __forceinline__ void store_head(const AppendParams& p, int half, int kind, int64_t block, int n_rows, bool anew, int h, int turn,
                            float4* cs, AppendCtl* ctl)
{
    const AppendJob& j = p.store;
    const int tid = threadIdx.x & (kAppHalf - 1);
    const int per_row = j.D / 16;
    const int turn_chunks = TURN ? p.ang.rot / 16 : 0;
    const int tile_rows = kAppTile / j.D;
    const int tiles = (n_rows + tile_rows - 1) / tile_rows;
    const T* x = static_cast<const T*>(j.x[kind]) + (int64_t)h * j.xs_h[kind];
    const uint32_t inf_bits = 0x7f800000u;
    float big = 0.f;
    float inv = 0.f;
    // f(values, raw values, row, item) for each of the block's items.  Items in flight per thread: as many as 64 registers hold.
    constexpr int UNR = TURN ? 2 : 4;
    auto walk = [&](auto&& f) {
        for (int tile = 0; tile < tiles; ++tile) {
            const int r0 = tile * tile_rows, items = min(tile_rows, n_rows - r0) * per_row;
            if (TURN && tiles > 1) {
                half_sync(half);  // nobody reads the old cosines any more
                fill_tile(p, cs, ctl, r0, min(tile_rows, n_rows - r0), tid, kAppHalf);
                half_sync(half);
            }
#pragma unroll UNR
            for (int i = tid; i < items; i += kAppHalf) {
                const int r = j.by_row.div(i), ch = i - r * per_row;
                const ItemPlace at = item_place(TURN, p.ang, ch);
                const T* src = x + (int64_t)ctl->tokens[r0 + r] * j.xs_t[kind];
                const uint4 va = *reinterpret_cast<const uint4*>(src + at.first), vb = *reinterpret_cast<const uint4*>(src + at.second);
                float a[8], b[8];
                item_values<T>(va, vb, TURN && ch < turn_chunks, cs + r * 4 * turn_chunks + ch, turn_chunks, p.ang.interleaved, a, b);
                f(a, b, va, vb, ctl->rows[r0 + r], ch);
            }
        }
    };
    if constexpr (CODES) {
        if constexpr (TURN) {
            walk([&](const float (&a)[8], const float (&b)[8], const uint4&, const uint4&, int, int) {
#pragma unroll
                for (int e = 0; e < 8; ++e) big = fmaxf(big, fmaxf(fabsf(a[e]), fabsf(b[e])));   // (NaN has no say)
            });
        } else {   // two values per instruction
            uint32_t two = 0;
            walk([&](const float (&)[8], const float (&)[8], const uint4& va, const uint4& vb, int, int) {
                two = Half2<T>::abs_max(Half2<T>::abs_max(Half2<T>::abs_max(Half2<T>::abs_max(two, va.x), va.y), va.z), va.w);
                two = Half2<T>::abs_max(Half2<T>::abs_max(Half2<T>::abs_max(Half2<T>::abs_max(two, vb.x), vb.y), vb.z), vb.w);
            });
            const float2 f = Half2<T>::to_float(two);
            big = fmaxf(f.x, f.y);
        }
        // The half's largest value -> scale (every thread computes the same); old codes are re-rounded if it grows.  The
        // words were last read two heads ago, on the other side of the previous head's barriers.
        uint32_t* word = &ctl->big[half][turn & 1];
        float* scale = j.scale[kind] + block * j.Hkv + h;
        const float old = anew ? 0.f : *scale;
        if (tid == 0) { word[0] = 0; word[2] = 0; }
        half_sync(half);  // (also: everybody has read the old scale)
        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
        if ((tid & 31) == 0) atomicMax(word, m);
        half_sync(half);
        uint32_t largest = word[0];
        const bool odd = largest >= inf_bits;
        if (odd) {        // an infinity among them: once more without
            float fin = 0.f;
            walk([&](const float (&a)[8], const float (&b)[8], const uint4&, const uint4&, int, int) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float ea = fabsf(a[e]), eb = fabsf(b[e]);
                    if (ea <= 3.402823466e38f) fin = fmaxf(fin, ea);
                    if (eb <= 3.402823466e38f) fin = fmaxf(fin, eb);
                }
            });
            atomicMax(word + 2, __float_as_uint(fin));
            half_sync(half);
            largest = word[2];
        }
        const float need = scale_for(__uint_as_float(largest));
        const float now = anew ? need : (old >= need ? old : need);  // (an old scale that is NaN is replaced)
        inv = inverse_scale(now);
        if (tid == 0) *scale = now;
        if (!anew && now != old) {
            const float ratio = old > 0.f ? old * inv : 0.f;
            uint8_t* base = static_cast<uint8_t*>(j.cache[kind]) + block * j.cs_b[kind] + (int64_t)h * j.cs_h[kind];
            for (int i = tid; i < j.BS * per_row; i += kAppHalf) {
                const int r = j.by_row.div(i);
                if (ctl->row_token[r] >= 0) continue;
                uint4* o = reinterpret_cast<uint4*>(base + (int64_t)r * j.cs_t[kind] + (i - r * per_row) * 16);
                const uint4 v = *o;
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t n[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float f[4];
                    from_e4m3x4(w[e], f);
#pragma unroll
                    for (int q = 0; q < 4; ++q) f[q] = ratio > 0.f ? f[q] * ratio : 0.f;
                    n[e] = to_e4m3x4<false>(f[0], f[1], f[2], f[3]);
                }
                *o = make_uint4(n[0], n[1], n[2], n[3]);
            }
        }
        auto put = [&](int row, int ch, const uint2& c0, const uint2& c1) {
            uint8_t* o = static_cast<uint8_t*>(j.cache[kind]) + block * j.cs_b[kind] + (int64_t)row * j.cs_t[kind] + (int64_t)h * j.cs_h[kind];
            const ItemPlace at = item_place(TURN, p.ang, ch);
            if (at.second == at.first + 8) {
                *reinterpret_cast<uint4*>(o + at.first) = make_uint4(c0.x, c0.y, c1.x, c1.y);
            } else {
                *reinterpret_cast<uint2*>(o + at.first) = c0;
                *reinterpret_cast<uint2*>(o + at.second) = c1;
            }
        };
        if (odd)
            walk([&](const float (&a)[8], const float (&b)[8], const uint4&, const uint4&, int row, int ch) { put(row, ch, codes8<true>(a, inv), codes8<true>(b, inv)); });
        else
            walk([&](const float (&a)[8], const float (&b)[8], const uint4&, const uint4&, int row, int ch) { put(row, ch, codes8<false>(a, inv), codes8<false>(b, inv)); });
    } else {
        walk([&](const float (&a)[8], const float (&b)[8], const uint4& wa, const uint4& wb, int row, int ch) {
            T* o = static_cast<T*>(j.cache[kind]) + block * j.cs_b[kind] + (int64_t)row * j.cs_t[kind] + (int64_t)h * j.cs_h[kind];
            const ItemPlace at = item_place(TURN, p.ang, ch);
            uint4 w;
            w.x = Half2<T>::from_float(a[0], a[1]); w.y = Half2<T>::from_float(a[2], a[3]);
            w.z = Half2<T>::from_float(a[4], a[5]); w.w = Half2<T>::from_float(a[6], a[7]);
            *reinterpret_cast<uint4*>(o + at.first) = ch < turn_chunks ? w : wa;
            w.x = Half2<T>::from_float(b[0], b[1]); w.y = Half2<T>::from_float(b[2], b[3]);
            w.z = Half2<T>::from_float(b[4], b[5]); w.w = Half2<T>::from_float(b[6], b[7]);
            *reinterpret_cast<uint4*>(o + at.second) = ch < turn_chunks ? w : wb;
        });
    }
}

template <typename T, bool CODES>
__device__ void append_chunk(const AppendParams& p, int64_t cta, float4* cs, AppendCtl* ctl)
{
    const AppendJob& j = p.store;
    const int64_t t0 = cta / j.head_tiles * j.chunk;
    const int h0 = (int)(cta % j.head_tiles) * j.heads_per_cta;
    const int nh = min(j.heads_per_cta, j.Hkv - h0);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t n_slots = j.NB * j.BS;
    const bool small = n_slots <= 0x7fffffff;   // slots divide by multiplication

    // candidates: tokens of the chunk whose predecessor in the list lies in another block
    if (tid == 0) { ctl->n_cand = 0; ctl->n_list = 0; }
    if (tid < 32) ctl->filter[tid] = 0;
    int64_t block = -1;
    bool starts = false;
    const int64_t t = t0 + tid;
    if (tid < j.chunk && t < j.T) {
        const int64_t s = load_index(j.slots, j.slot_is_int64, t);
        if (s >= 0 && s < n_slots) {
            block = s / j.BS;
            const int64_t before = t > 0 ? load_index(j.slots, j.slot_is_int64, t - 1) : -1;
            starts = !(before >= 0 && before < n_slots && before / j.BS == block);
        }
    }
    const uint32_t votes = __ballot_sync(0xffffffffu, starts);
    if (lane == 0 && warp < kAppMaxChunk / 32) ctl->warp_count[warp] = __popc(votes);
    __syncthreads();
    if (starts) {
        int at = __popc(votes & ((1u << lane) - 1));
        for (int w = 0; w < warp; ++w) at += ctl->warp_count[w];
        ctl->cand_block[at] = block;
        ctl->cand_token[at] = (int)t;
        ctl->lead[at] = 1;
        const uint32_t b = filter_bit(block);
        atomicOr(&ctl->filter[b >> 5], 1u << (b & 31));
        atomicAdd(&ctl->n_cand, 1);
    }
    __syncthreads();
    const int n_cand = ctl->n_cand;
    if (n_cand == 0) return;

    // the walk: every token of a candidate's block, and whether an earlier token makes another CTA (or candidate) the owner;
    // eight slots at a time, since each is a round trip to L2
    constexpr int kWalk = 8;
    for (int64_t u0 = tid; u0 < j.T; u0 += kWalk * 2 * kAppHalf) {
        int64_t slot[kWalk];
#pragma unroll
        for (int k = 0; k < kWalk; ++k) {
            const int64_t u = u0 + k * 2 * kAppHalf;
            slot[k] = u < j.T ? load_index(j.slots, j.slot_is_int64, u) : -1;
        }
#pragma unroll
        for (int k = 0; k < kWalk; ++k) {
            if (slot[k] < 0 || slot[k] >= n_slots) continue;
            const int64_t b = small ? (int64_t)j.by_block.div((int)slot[k]) : slot[k] / j.BS;
            const uint32_t bit = filter_bit(b);
            if (!((ctl->filter[bit >> 5] >> (bit & 31)) & 1u)) continue;
            const int64_t u = u0 + k * 2 * kAppHalf;
            for (int c = 0; c < n_cand; ++c) {
                if (ctl->cand_block[c] != b) continue;
                if (u < ctl->cand_token[c]) { ctl->lead[c] = 0; continue; }
                const int at = atomicAdd(&ctl->n_list, 1);
                if (at < kAppList) { ctl->list_cand[at] = c; ctl->list_token[at] = (int)u; }
            }
        }
    }
    __syncthreads();
    const int n_list = ctl->n_list;

    for (int c = 0; c < n_cand; ++c) {
        if (!ctl->lead[c]) continue;  // (the same for all threads)
        const int64_t b = ctl->cand_block[c];
        for (int r = tid; r < j.BS; r += blockDim.x) ctl->row_token[r] = -1;
        __syncthreads();
        if (n_list <= kAppList) {
            for (int i = tid; i < n_list; i += blockDim.x) {
                if (ctl->list_cand[i] != c) continue;
                const int u = ctl->list_token[i];
                atomicMax(&ctl->row_token[(int)(load_index(j.slots, j.slot_is_int64, u) - b * j.BS)], u);
            }
        } else {
            for (int64_t u = tid; u < j.T; u += blockDim.x) {
                const int64_t s = load_index(j.slots, j.slot_is_int64, u);
                if (s >= 0 && s < n_slots && s / j.BS == b) atomicMax(&ctl->row_token[(int)(s - b * j.BS)], (int)u);
            }
        }
        __syncthreads();
        if (warp == 0) {
            int n = 0;
            for (int r0 = 0; r0 < j.BS; r0 += 32) {
                const bool on = r0 + lane < j.BS && ctl->row_token[r0 + lane] >= 0;
                const uint32_t m = __ballot_sync(0xffffffffu, on);
                if (on) {
                    const int at = n + __popc(m & ((1u << lane) - 1));
                    ctl->rows[at] = r0 + lane;
                    ctl->tokens[at] = ctl->row_token[r0 + lane];
                }
                n += __popc(m);
            }
            if (lane == 0) ctl->n_rows = n;
        }
        __syncthreads();
        if (p.ang.inv_freq != nullptr && ctl->n_rows <= kAppTile / j.D) {
            fill_tile(p, cs, ctl, 0, ctl->n_rows, tid, 2 * kAppHalf);
            __syncthreads();
        }
        // Keys take longer than values, by their rotation: the halves take them in turn.  Not where the table of cosines is
        // filled tile by tile, by the half that holds the keys.
        const int half = tid / kAppHalf;
        const bool swap = ctl->n_rows <= kAppTile / j.D;
        for (int hi = 0; hi < nh; ++hi) {
            const int kind = swap ? (half + hi) & 1 : half;
            if (kind == 0 && p.ang.inv_freq != nullptr)
                store_head<T, CODES, true>(p, half, kind, b, ctl->n_rows, ctl->row_token[0] >= 0, h0 + hi, hi, cs, ctl);
            else
                store_head<T, CODES, false>(p, half, kind, b, ctl->n_rows, ctl->row_token[0] >= 0, h0 + hi, hi, cs, ctl);
        }
        __syncthreads();
    }
}

template <typename T, bool CODES>
__global__ void __launch_bounds__(2 * kAppHalf, 2) kv_append_kernel(const __grid_constant__ AppendParams p)
{
    extern __shared__ float4 s_dyn[];
    int64_t cta = blockIdx.x;
    // the store's CTAs come first: they take longest (spread among the others: 180 -> 253 us)
    const int64_t n_store = (p.store.T + p.store.chunk - 1) / p.store.chunk * p.store.head_tiles;
    if (cta < n_store) {
        AppendCtl* ctl = reinterpret_cast<AppendCtl*>(s_dyn);
        append_chunk<T, CODES>(p, cta, s_dyn + (sizeof(AppendCtl) + 15) / 16, ctl);
        return;
    }
    cta -= n_store;
    const int k = cta < p.rot_ctas[0] ? 0 : 1;
    if (k == 1) cta -= p.rot_ctas[0];
    if (p.rot_vector[k]) rotate_tile<T, 2 * kAppHalf>(p.rot[k], p.ang, cta, s_dyn);
    else rotate_scalar<T>(p.rot[k], p.ang, cta * 2 * kAppHalf + threadIdx.x, p.rot_ctas[k] * 2 * kAppHalf);
}

template <typename T, bool CODES>
static int launch_append(AppendParams& p, cudaStream_t st)
{
    AppendJob& j = p.store;
    const int sms = device_sms();
    // Chunk: one token while that leaves at most eight CTAs per SM (a decode step: one owner per CTA), up to 128 tokens
    // (one walk of the slot list for a whole block of 128).  Heads per CTA: one, doubled while the grid has more than three
    // CTAs per SM, since every CTA repeats the walk and the cosines (measured for the call above: 180 us; up to six 202, twelve 242).
    int64_t chunk = (j.T * j.Hkv + (int64_t)sms * 8 - 1) / ((int64_t)sms * 8);
    j.chunk = (int)(chunk < 1 ? 1 : chunk > kAppMaxChunk ? kAppMaxChunk : chunk);
    const int64_t chunks = (j.T + j.chunk - 1) / j.chunk;
    j.heads_per_cta = 1;
    while (j.heads_per_cta < j.Hkv && chunks * ((j.Hkv + j.heads_per_cta - 1) / j.heads_per_cta) > (int64_t)sms * 3) j.heads_per_cta *= 2;
    j.head_tiles = (j.Hkv + j.heads_per_cta - 1) / j.heads_per_cta;
    int64_t ctas = chunks * j.head_tiles;
    const int tile_rows = kAppTile / j.D < j.BS ? kAppTile / j.D : j.BS;
    size_t smem = (sizeof(AppendCtl) + 15) / 16 * 16;
    if (p.ang.inv_freq) smem += (size_t)tile_rows * (p.ang.rot / 16) * 64;
    for (int k = 0; k < 2; ++k) {
        RotaryJob& r = p.rot[k];
        p.rot_ctas[k] = 0;
        if (r.T == 0 || r.H == 0) continue;
        p.rot_vector[k] = rotary_vector_ok(r, p.ang.rot);
        if (p.rot_vector[k]) {
            plan_rotary(r, p.ang.rot, sms);
            p.rot_ctas[k] = rotary_ctas(r);
            const size_t need = rotary_smem(r, p.ang.rot);
            if (need > smem) smem = need;
        } else {
            const int64_t n = (r.T * r.H * (r.D - p.ang.rot / 2) + 2 * kAppHalf - 1) / (2 * kAppHalf);
            p.rot_ctas[k] = n < (int64_t)sms * 8 ? n : (int64_t)sms * 8;
        }
        ctas += p.rot_ctas[k];
    }
    if (ctas > 0x7FFFFFFF) return UCMR_ERR_UNSUPPORTED;
    cudaError_t e = cudaFuncSetAttribute(kv_append_kernel<T, CODES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) { note_cuda_error(e); (void)cudaGetLastError(); return UCMR_ERR_LAUNCH; }
    return launch_kernel(kv_append_kernel<T, CODES>, dim3((unsigned)ctas), dim3(2 * kAppHalf), smem, st, p);
}

}  // namespace ucmr

extern "C" int ucmr_kv_append(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                              int64_t v_stride_h, int64_t T, int Hkv, int D, int dtype, const void* slot_mapping,
                              int slot_is_int64, void* k_cache, int64_t kc_stride_block, int64_t kc_stride_t,
                              int64_t kc_stride_h, void* v_cache, int64_t vc_stride_block, int64_t vc_stride_t,
                              int64_t vc_stride_h, int64_t NB, int BS, int cache_dtype, float* k_scale, float* v_scale,
                              const void* positions, int pos_is_int64, const double* inv_freq, int rotary_dim,
                              int interleaved, float mscale, const void* q, int Hq, int64_t q_stride_t, int64_t q_stride_h,
                              void* q_out, int64_t qo_stride_t, int64_t qo_stride_h, void* k_out, int64_t ko_stride_t,
                              int64_t ko_stride_h, void* stream)
{
    using namespace ucmr;
    if (T < 0 || Hkv <= 0 || D <= 0 || NB < 0 || BS <= 0 || (q && Hq <= 0)) return UCMR_ERR_BAD_ARG;
    if (dtype != UCMR_BF16 && dtype != UCMR_FP16) return UCMR_ERR_UNSUPPORTED;
    if (cache_dtype != dtype && cache_dtype != UCMR_E4M3) return UCMR_ERR_UNSUPPORTED;
    if (cache_dtype == UCMR_E4M3 ? (!k_scale || !v_scale) : (k_scale || v_scale)) return UCMR_ERR_BAD_ARG;
    if (inv_freq && (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > D)) return UCMR_ERR_BAD_ARG;
    if (!inv_freq && (q || k_out)) return UCMR_ERR_BAD_ARG;
    if (D % 16 != 0 || D > 512 || BS > kAppMaxBlock || (inv_freq && rotary_dim % 16 != 0)) return UCMR_ERR_UNSUPPORTED;
    if (T > kAppMaxTokens || NB * (int64_t)BS > ((int64_t)1 << 46)) return UCMR_ERR_UNSUPPORTED;
    if (T == 0) return UCMR_OK;
    if (!k || !v || !slot_mapping || !k_cache || !v_cache || (inv_freq && !positions) || (q && !q_out) || k_out == k) return UCMR_ERR_BAD_ARG;
    // whole 16-byte vectors of every row, in and out
    const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_cache) |
                           reinterpret_cast<uintptr_t>(v_cache);
    const int64_t in = k_stride_t | k_stride_h | v_stride_t | v_stride_h;
    const int64_t cs = kc_stride_block | kc_stride_t | kc_stride_h | vc_stride_block | vc_stride_t | vc_stride_h;
    if (bits % 16 != 0 || in % 8 != 0 || cs % (cache_dtype == UCMR_E4M3 ? 16 : 8) != 0) return UCMR_ERR_UNSUPPORTED;

    AppendParams p{};
    p.ang.inv_freq = inv_freq; p.ang.positions = positions; p.ang.pos_is_int64 = pos_is_int64; p.ang.rot = inv_freq ? rotary_dim : 0;
    p.ang.interleaved = interleaved; p.ang.mscale = mscale; p.ang.transpose = 0;
    AppendJob& j = p.store;
    j.x[0] = k; j.xs_t[0] = k_stride_t; j.xs_h[0] = k_stride_h;
    j.x[1] = v; j.xs_t[1] = v_stride_t; j.xs_h[1] = v_stride_h;
    j.cache[0] = k_cache; j.cs_b[0] = kc_stride_block; j.cs_t[0] = kc_stride_t; j.cs_h[0] = kc_stride_h;
    j.cache[1] = v_cache; j.cs_b[1] = vc_stride_block; j.cs_t[1] = vc_stride_t; j.cs_h[1] = vc_stride_h;
    j.scale[0] = k_scale; j.scale[1] = v_scale;
    j.by_row = FastDiv::by((uint32_t)(D / 16)); j.by_block = FastDiv::by((uint32_t)BS); j.slots = slot_mapping; j.slot_is_int64 = slot_is_int64; j.T = T; j.NB = NB; j.BS = BS; j.Hkv = Hkv; j.D = D;
    if (q) {
        RotaryJob& r = p.rot[0];
        r.x = q; r.out = q_out; r.T = T; r.H = Hq; r.D = D;
        r.xs_t = q_stride_t; r.xs_h = q_stride_h; r.os_t = qo_stride_t; r.os_h = qo_stride_h;
    }
    if (k_out) {
        RotaryJob& r = p.rot[1];
        r.x = k; r.out = k_out; r.T = T; r.H = Hkv; r.D = D;
        r.xs_t = k_stride_t; r.xs_h = k_stride_h; r.os_t = ko_stride_t; r.os_h = ko_stride_h;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cache_dtype == UCMR_E4M3)
        return dtype == UCMR_BF16 ? launch_append<__nv_bfloat16, true>(p, st) : launch_append<__half, true>(p, st);
    return dtype == UCMR_BF16 ? launch_append<__nv_bfloat16, false>(p, st) : launch_append<__half, false>(p, st);
}
