// Attention over the paged KV cache (sm_100a): out = softmax(scale * q k^T) v over the tokens of the blocks that a table
// lists, for decode steps, speculative verification and short prefills.  Cache of 16-bit values, or of e4m3 codes with a
// scale per (block, kv head).
//
// Work.  An item is (request, row tile, kv head): the G query heads of a kv head times the request's query tokens give
// rows; NT * 8 of them share one pass over the keys.  Its tokens are cut into units of 128.  All units of all items form
// one line, which is divided evenly over the CTAs (two per SM): ragged batches balance, and one long request is split
// over the whole GPU.  A CTA that has only a part of an item leaves (max, sum, unnormalised rows) in its slot of the
// workspace; the last of an item's CTAs to arrive adds the parts up, in the order of the tokens: results do not depend
// on timing.  HBM-bound for up to 16 rows: the keys and values are read once.
//
// A unit is eight warps times 16 tokens, and the warps do not wait for one another.  Each has a ring of stages in shared
// memory that its own lanes fill with 16-byte asynchronous copies; a lane reads back only what it copied itself, so a
// stage needs no barrier, and block ids, scales and tails are handled per token: any block size, any strides.
//   S^T = K Q^T: tokens are the 16 rows of mma.m16n8k16, query rows its 8 columns.  The order in which the products run
//     over the head dimension is free, so each lane takes 16 consecutive bytes of a key (4 lanes per key), converts them
//     and has its fragments; the queries are read in the same order.
//   O^T += V^T P^T: the head dimension is the 16 rows, again in a free order: each lane takes D/8 consecutive values of four
//     tokens, and interleaves the tokens two by two for its fragments.  P^T is S^T's fragment, transposed by movmatrix.
// mma.sync serves here because the rows are few: 16 x 8 tiles waste nothing, and the tensor work is a fifth of what the
// legacy path can do while the memory system is saturated.
//
// Numerics.  e4m3 codes become fp16 exactly; queries become fp16 after a power of two per row has brought them to at most
// 2 (bf16 -> fp16 is then exact but for values below 2^-24 of the row's largest).  Scores, softmax and rows are float32; the key scale and the softmax scale are applied to
// the float32 score.  The probability that multiplies V is rounded to fp16 (half a step: 2^-11) with the value scale
// folded in, counted from 2^(14 - E), E the exponent of the largest value scale so far: the largest product is 2^14, so
// probabilities down to 2^-28 of the largest keep all bits and those below 2^-39 are dropped.  A bf16 cache uses bf16 operands
// (probabilities rounded by 2^-8), an fp16 cache fp16 ones.
#include "paged_attention.cuh"

namespace ucmr {

int device_sms();
int attention_tiles(const AttnParams& p, int D, int dtype, int cache_dtype, cudaStream_t st);  // paged_prefill.cu

enum { kBf16 = 0, kF16 = 1, kE4m3 = 2 };

constexpr int kDecWarps = 8;
constexpr int kDecUnit = kDecWarps * 16;
constexpr float kShift = 14.f;  // see "Numerics"

template <int D, int C>
struct DecShape {
    static constexpr int kEs = C == kE4m3 ? 1 : 2;          // bytes per cached value
    static constexpr int kKPieces = D * kEs / 64;           // 16-byte pieces of a key per lane
    static constexpr int kVBytes = D * kEs / 8;             // bytes of a value row per lane
    static constexpr int kVCopy = kVBytes < 16 ? kVBytes : 16;
    static constexpr int kVPieces = kVBytes / kVCopy;
    static constexpr int kKStage = 2 * kKPieces * 32 * 16;
    static constexpr int kVStage = 4 * kVPieces * 32 * kVCopy;
    static constexpr int kScaleStage = 32 * 4 + 16;         // 16 key scales, 16 value scales, mask of live tokens
    static constexpr int kStage = kKStage + kVStage + kScaleStage;
    static constexpr int kKSteps = D / 16;
    static constexpr int kMTiles = D / 16;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(live ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int C>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (C == kBf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
    return r;
}

__device__ __forceinline__ float unpack_16(uint32_t v, int high, bool bf16)
{
    const uint16_t h = (uint16_t)(high ? v >> 16 : v);
    return bf16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}

template <int C>
__device__ __forceinline__ uint32_t pack_p(float lo, float hi)
{
    if constexpr (C == kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(h);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(h);
    }
}

// One of the CTA's stretches: units [first, last) of one item.
struct Segment {
    int b, rt, h, first, last, units;
    AttnRequest r;
};

template <int D, int C, int NT, int STAGES>
struct DecShared {
    alignas(16) unsigned char ring[kDecWarps][STAGES][DecShape<D, C>::kStage];
    // (a warp's rows take the place of its own ring once its copies have landed)
    static_assert(STAGES * DecShape<D, C>::kStage >= NT * 8 * D * 4, "rows do not fit the ring");
    float m[kDecWarps][NT * 8], l[kDecWarps][NT * 8];
    float weight[kDecWarps][NT * 8];
    float row_m[NT * 8], row_l[NT * 8];
    unsigned long long sums[kDecWarps];
    unsigned long long start_units;
    int start_b;
    int last;
};

template <int D, int C, int NT, int STAGES, typename QT>
__global__ void __launch_bounds__(kDecWarps * 32) decode_kernel(const __grid_constant__ AttnParams p)
{
    using Sh = DecShape<D, C>;
    using Smem = DecShared<D, C, NT, STAGES>;
    extern __shared__ __align__(16) unsigned char s_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(s_raw);
    constexpr int R = NT * 8;
    auto rows_of = [&](int w) { return reinterpret_cast<float*>(&sm.ring[w][0][0]); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    constexpr bool kQBf16 = sizeof(QT) == 2 && __is_same(QT, __nv_bfloat16);

    // ---- this CTA's stretch of the line of units -------------------------------------------------------------
    auto units_of = [&](const AttnRequest& r) { return (r.len + kDecUnit - 1) / kDecUnit; };
    auto tiles_of = [&](const AttnRequest& r) { return (int)(((int64_t)r.nq * p.G + R - 1) / R); };
    // (an item without tokens still takes one unit: its rows are written as empty)
    auto line_of = [&](int b) -> unsigned long long {
        const AttnRequest r = attn_request(p, b);
        return (unsigned long long)max(1, units_of(r)) * (unsigned)tiles_of(r) * (unsigned)p.Hkv;
    };
    const int per = (p.B + kDecWarps * 32 - 1) / (kDecWarps * 32);
    unsigned long long mine = 0;
    for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) mine += line_of(b);
    unsigned long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) sm.sums[warp] = before;
    __syncthreads();
    unsigned long long total = 0, offset = 0;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
        if (w < warp) offset += sm.sums[w];
        total += sm.sums[w];
    }
    before += offset - mine;
    const unsigned long long n_cta = min((unsigned long long)gridDim.x, total);
    if (blockIdx.x >= n_cta) return;
    const unsigned long long u0 = blockIdx.x * total / n_cta, u1 = (blockIdx.x + 1) * total / n_cta;
    if (before <= u0 && u0 < before + mine) {
        unsigned long long at = before;
        for (int b = tid * per; b < p.B; ++b) {
            const unsigned long long n = line_of(b);
            if (u0 < at + n) { sm.start_b = b; sm.start_units = at; break; }
            at += n;
        }
    }
    __syncthreads();
    int b = sm.start_b;
    unsigned long long b_first = sm.start_units;  // line position of request b

    const uint32_t ring = smem_u32(&sm.ring[warp][0][0]);
    const float inf = __uint_as_float(0x7f800000u);

    for (unsigned long long u = u0; u < u1;) {
        // ---- the segment that starts at u ---------------------------------------------------------------------
        Segment s;
        for (;;) {
            if (b >= p.B) return;  // (lengths that changed under the kernel)
            s.r = attn_request(p, b);
            s.units = max(1, units_of(s.r));
            const unsigned long long n = (unsigned long long)s.units * (unsigned)tiles_of(s.r) * (unsigned)p.Hkv;
            if (u < b_first + n) break;
            b_first += n;
            ++b;
        }
        const unsigned long long in_b = u - b_first;
        const int item = (int)(in_b / s.units);
        s.b = b;
        s.h = item % p.Hkv;
        s.rt = item / p.Hkv;
        s.first = (int)(in_b - (unsigned long long)item * s.units);
        const unsigned long long item_first = u - s.first;
        s.last = (int)min((unsigned long long)s.units, u1 - item_first);
        const int row0 = s.rt * R, n_rows = s.r.nq * p.G;  // rows of the request; this tile holds [row0, row0 + R)

        // ---- queries: fragments of the second operand, row n = g of each group of eight --------------------------------
        uint32_t qf[NT][Sh::kKSteps][2];
        float qmul[NT][2];  // score factor of the columns 2t and 2t+1
        int limit[NT][2];
        int max_limit = 0, min_limit = 0x7fffffff;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = row0 + nt * 8 + g;
            const bool live = row < n_rows;
            const QT* qr = static_cast<const QT*>(p.q);
            if (live) qr += (int64_t)(s.r.q0 + row / p.G) * p.qs_t + (int64_t)(s.h * p.G + row % p.G) * p.qs_h;
            uint32_t raw[Sh::kKSteps][2];
#pragma unroll
            for (int ks = 0; ks < Sh::kKSteps; ++ks) {
                // product step ks takes four elements of each lane of the quad: word ks%4 (e4m3) or words 2*(ks%2) and
                // 2*(ks%2)+1 (16 bit) of 16-byte piece ks/4 or ks/2
                constexpr int kPerPiece = C == kE4m3 ? 4 : 2;
                const int d = (ks / kPerPiece) * (64 / Sh::kEs) + t * (16 / Sh::kEs) + (ks % kPerPiece) * 4;
                raw[ks][0] = raw[ks][1] = 0;
                if (live) {
                    const uint2 v = *reinterpret_cast<const uint2*>(qr + d);
                    raw[ks][0] = v.x;
                    raw[ks][1] = v.y;
                }
            }
            float mul = 1.f;
            if constexpr (C == kE4m3) {
                uint32_t big = 0;  // largest finite magnitude of the row, as float bits
#pragma unroll
                for (int ks = 0; ks < Sh::kKSteps; ++ks)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t v = __float_as_uint(fabsf(unpack_16(raw[ks][i >> 1], i & 1, kQBf16)));
                        if (v < 0x7f800000u) big = max(big, v);
                    }
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                // 2^e <= big < 2^(e+1): the row times 2^-e lies below 2
                const int e = big == 0 ? 0 : max(-125, min(125, (int)(big >> 23) - 127));
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                mul = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int ks = 0; ks < Sh::kKSteps; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        qf[nt][ks][i] = pack_p<kF16>(unpack_16(raw[ks][i], 0, kQBf16) * down, unpack_16(raw[ks][i], 1, kQBf16) * down);
            } else {
#pragma unroll
                for (int ks = 0; ks < Sh::kKSteps; ++ks) { qf[nt][ks][0] = raw[ks][0]; qf[nt][ks][1] = raw[ks][1]; }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                qmul[nt][i] = __shfl_sync(0xffffffffu, mul, 8 * t + 4 * i) * p.scale_log2;
                const int r2 = row0 + nt * 8 + 2 * t + i;
                limit[nt][i] = r2 < n_rows ? attn_limit(p, s.r, r2 / p.G) : 0;
            }
        }
        {
            const int first_row = row0 / p.G, last_row = min(n_rows, row0 + R) - 1;
            if (last_row >= row0) {
                max_limit = attn_limit(p, s.r, last_row / p.G);
                min_limit = attn_limit(p, s.r, first_row);
            }
        }

        float o[NT][Sh::kMTiles][4];
        float m[NT][2], l[NT][2];
        int vexp = -200;  // E of "Numerics"; o is counted from 2^(E - 14)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < Sh::kMTiles; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
            m[nt][0] = m[nt][1] = -inf;
            l[nt][0] = l[nt][1] = 0.f;
        }

        // ---- tokens -----------------------------------------------------------------------------------------------
        const int32_t* table = p.table + (int64_t)s.b * p.bt_b + (int64_t)s.h * p.bt_h;
        const int n_tiles = s.last - s.first;  // tiles of this warp: one per unit
        auto token_of = [&](int i) { return (s.first + i) * kDecUnit + warp * 16 + (lane & 15); };
        auto block_of = [&](int i) {
            const int tok = token_of(i);
            return i < n_tiles && tok < max_limit ? table[p.by_block.div(tok)] : -1;
        };
        auto issue = [&](int i, int blk) {
            const uint32_t stage = ring + (uint32_t)(i % STAGES) * Sh::kStage;
            const int tok = token_of(i);
            const bool in = i < n_tiles && tok < max_limit;
            bool live = in && blk >= 0 && blk < p.NB;
            if (in && !live) flag_status(p.status, UCMR_DEV_BAD_BLOCK_ID);
            const int row = tok - p.by_block.div(tok) * p.BS;
            const int64_t ko = live ? blk * p.cs_b[0] + row * p.cs_t[0] + s.h * p.cs_h[0] : 0;
            const int64_t vo = live ? blk * p.cs_b[1] + row * p.cs_t[1] + s.h * p.cs_h[1] : 0;
            const uint32_t mask = __ballot_sync(0xffffffffu, live) & 0xffffu;
            const char* kb = static_cast<const char*>(p.cache[0]);
            const char* vb = static_cast<const char*>(p.cache[1]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const char* src = kb + __shfl_sync(0xffffffffu, ko, g + 8 * half) + t * 16;
                const bool on = (mask >> (g + 8 * half)) & 1u;
#pragma unroll
                for (int c = 0; c < Sh::kKPieces; ++c)
                    cp_async16(stage + ((half * Sh::kKPieces + c) * 32 + lane) * 16, on ? src + c * 64 : kb, on);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int tk = 2 * t + (k & 1) + 8 * (k >> 1);
                const char* src = vb + __shfl_sync(0xffffffffu, vo, tk) + g * Sh::kVBytes;
                const bool on = (mask >> tk) & 1u;
#pragma unroll
                for (int c = 0; c < Sh::kVPieces; ++c) {
                    const uint32_t dst = stage + Sh::kKStage + ((k * Sh::kVPieces + c) * 32 + lane) * Sh::kVCopy;
                    if constexpr (Sh::kVCopy == 16) cp_async16(dst, on ? src + c * 16 : vb, on);
                    else cp_async8(dst, on ? src : vb, on);
                }
            }
            if constexpr (C == kE4m3) {
                const float* sc = p.scale[lane >> 4];
                cp_async4(stage + Sh::kKStage + Sh::kVStage + lane * 4, live ? sc + (int64_t)blk * p.Hkv + s.h : sc, live);
            }
            if (lane == 0) *reinterpret_cast<uint32_t*>(s_raw + (stage - smem_u32(s_raw)) + Sh::kKStage + Sh::kVStage + 128) = mask;
        };

        int next = block_of(0);
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            const int blk = next;
            next = block_of(i + 1);
            if (i < n_tiles) issue(i, blk);
            cp_async_commit();
        }
        for (int i = 0; i < n_tiles; ++i) {
            {
                const int blk = next;
                next = block_of(i + STAGES);
                __syncwarp();  // every lane is done with the stage that is filled now
                if (i + STAGES - 1 < n_tiles) issue(i + STAGES - 1, blk);
                cp_async_commit();
            }
            cp_async_wait<STAGES - 1>();
            __syncwarp();  // scales and mask come from other lanes
            const unsigned char* st = &sm.ring[warp][i % STAGES][0];
            const int tok0 = (s.first + i) * kDecUnit + warp * 16;
            const uint32_t mask = *reinterpret_cast<const uint32_t*>(st + Sh::kKStage + Sh::kVStage + 128);
            if (mask == 0) continue;

            // scores of tokens g and g + 8
            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
            for (int c = 0; c < Sh::kKPieces; ++c) {
                const uint4 lo = *reinterpret_cast<const uint4*>(st + (c * 32 + lane) * 16);
                const uint4 hi = *reinterpret_cast<const uint4*>(st + ((Sh::kKPieces + c) * 32 + lane) * 16);
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
                if constexpr (C == kE4m3) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = e4m3x2_to_f16x2(wl[w]), a2 = e4m3x2_to_f16x2(wl[w] >> 16);
                        const uint32_t a1 = e4m3x2_to_f16x2(wh[w]), a3 = e4m3x2_to_f16x2(wh[w] >> 16);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816<C>(sc[nt], a0, a1, a2, a3, qf[nt][c * 4 + w][0], qf[nt][c * 4 + w][1]);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_16816<C>(sc[nt], wl[2 * w], wh[2 * w], wl[2 * w + 1], wh[2 * w + 1], qf[nt][c * 2 + w][0], qf[nt][c * 2 + w][1]);
                }
            }
            float vfac0 = C == kBf16 ? 1.f : 16384.f, vfac1 = vfac0;
            float ks0 = 1.f, ks1 = 1.f;
            float vdown = 1.f;
            if constexpr (C == kE4m3) {
                const float* f = reinterpret_cast<const float*>(st + Sh::kKStage + Sh::kVStage);
                ks0 = f[g];
                ks1 = f[g + 8];
                const float v0 = f[16 + g], v1 = f[24 + g];
                const uint32_t big = __reduce_max_sync(0xffffffffu, max(__float_as_uint(fabsf(v0)), __float_as_uint(fabsf(v1))));
                const int e = max(-100, min(128, (int)(big >> 23) - 126));  // every scale is below 2^e
                if (e > vexp) {
                    vdown = vexp == -200 ? 0.f : exp2_fast((float)(vexp - e));
                    vexp = e;
                }
                const float up = exp2_fast(kShift - (float)vexp);  // a power of two
                vfac0 = v0 * up;
                vfac1 = v1 * up;
            }
            const bool edge = mask != 0xffffu || tok0 + 16 > min_limit;
            bool grown = vdown != 1.f;
            float alpha[NT][2];
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float x[4];
                x[0] = sc[nt][0] * (ks0 * qmul[nt][0]);
                x[1] = sc[nt][1] * (ks0 * qmul[nt][1]);
                x[2] = sc[nt][2] * (ks1 * qmul[nt][0]);
                x[3] = sc[nt][3] * (ks1 * qmul[nt][1]);
                if (edge) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int tk = g + 8 * (c >> 1);
                        if (!((mask >> tk) & 1u) || tok0 + tk >= limit[nt][c & 1]) x[c] = -inf;
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = fmaxf(x[c], x[c + 2]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    alpha[nt][c] = 1.f;
                    if (top > m[nt][c]) {
                        alpha[nt][c] = exp2_fast(m[nt][c] - top);  // (0 from -inf)
                        m[nt][c] = top;
                        grown = true;
                    }
                    const float ref = m[nt][c] == -inf ? 0.f : m[nt][c];
                    const float p0 = exp2_fast(x[c] - ref), p1 = exp2_fast(x[c + 2] - ref);
                    l[nt][c] = l[nt][c] * alpha[nt][c] + (p0 + p1);
                    x[c] = p0 * vfac0;
                    x[c + 2] = p1 * vfac1;
                }
                pf[nt][0] = transpose_8x8(pack_p<C == kBf16 ? kBf16 : kF16>(x[0], x[1]));
                pf[nt][1] = transpose_8x8(pack_p<C == kBf16 ? kBf16 : kF16>(x[2], x[3]));
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f0 = alpha[nt][0] * vdown, f1 = alpha[nt][1] * vdown;
#pragma unroll
                    for (int k = 0; k < Sh::kMTiles; ++k) {
                        o[nt][k][0] *= f0; o[nt][k][1] *= f1;
                        o[nt][k][2] *= f0; o[nt][k][3] *= f1;
                    }
                }
            }
            // values: D/8 consecutive ones of tokens 2t, 2t+1, 2t+8, 2t+9
            const unsigned char* sv = st + Sh::kKStage;
            constexpr int W = Sh::kVBytes / 4;
            uint32_t vw[4][W];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (Sh::kVCopy == 16) {
#pragma unroll
                    for (int c = 0; c < Sh::kVPieces; ++c) {
                        const uint4 v = *reinterpret_cast<const uint4*>(sv + ((k * Sh::kVPieces + c) * 32 + lane) * 16);
                        vw[k][c * 4] = v.x; vw[k][c * 4 + 1] = v.y; vw[k][c * 4 + 2] = v.z; vw[k][c * 4 + 3] = v.w;
                    }
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(sv + (k * 32 + lane) * 8);
                    vw[k][0] = v.x;
                    vw[k][1] = v.y;
                }
            }
            if (edge && tok0 + 16 > min_limit && min_limit < max_limit) {
                // Some rows see these tokens and some do not: a value that is not finite must not reach the latter as
                // 0 * NaN.  It is taken out of the product and added by itself to the rows that see it.
                bool odd = false;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        if constexpr (C == kE4m3) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (((vw[k][w] >> (8 * e)) & 0x7fu) == 0x7fu) { vw[k][w] &= ~(0xffu << (8 * e)); odd = true; }
                        } else {
                            constexpr uint32_t kExp = C == kBf16 ? 0x7f80u : 0x7c00u;
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (((vw[k][w] >> (16 * e)) & kExp) == kExp) { vw[k][w] &= ~(0xffffu << (16 * e)); odd = true; }
                        }
                    }
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
                    for (int tk = 0; tk < 16; ++tk) {
                        const int k = (tk & 1) + 2 * (tk >> 3), owner = (g << 2) | ((tk & 7) >> 1);
#pragma unroll
                        for (int d = 0; d < D / 8; ++d) {
                            const int byte = d * Sh::kEs;
                            const unsigned char* at = sv + ((k * Sh::kVPieces + byte / Sh::kVCopy) * 32 + owner) * Sh::kVCopy + byte % Sh::kVCopy;
                            float v = 0.f;
                            if constexpr (C == kE4m3) {
                                if ((*at & 0x7fu) == 0x7fu) v = __uint_as_float(0x7fffffffu);
                            } else {
                                const float x = unpack_16(*reinterpret_cast<const uint16_t*>(at), 0, C == kBf16);
                                if (!(fabsf(x) <= 3.402823466e38f)) v = x;
                            }
                            if (v == 0.f) continue;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 2; ++c)
                                    if (((mask >> tk) & 1u) && tok0 + tk < limit[nt][c]) o[nt][d / 2][(d & 1) * 2 + c] += v;
                        }
                    }
                }
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if constexpr (C == kE4m3) {
                    // bytes of two tokens side by side: (token 0, token 1) of values 4w, 4w+1 | 4w+2, 4w+3
                    const uint32_t x0 = __byte_perm(vw[0][w], vw[1][w], 0x5140), x1 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
                    const uint32_t y0 = __byte_perm(vw[2][w], vw[3][w], 0x5140), y1 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
                    const uint32_t a0 = e4m3x2_to_f16x2(x0), a1 = e4m3x2_to_f16x2(x0 >> 16);
                    const uint32_t a2 = e4m3x2_to_f16x2(y0), a3 = e4m3x2_to_f16x2(y0 >> 16);
                    const uint32_t b0 = e4m3x2_to_f16x2(x1), b1 = e4m3x2_to_f16x2(x1 >> 16);
                    const uint32_t b2 = e4m3x2_to_f16x2(y1), b3 = e4m3x2_to_f16x2(y1 >> 16);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16816<C>(o[nt][2 * w], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                        mma_16816<C>(o[nt][2 * w + 1], b0, b1, b2, b3, pf[nt][0], pf[nt][1]);
                    }
                } else {
                    const uint32_t a0 = __byte_perm(vw[0][w], vw[1][w], 0x5410), a1 = __byte_perm(vw[0][w], vw[1][w], 0x7632);
                    const uint32_t a2 = __byte_perm(vw[2][w], vw[3][w], 0x5410), a3 = __byte_perm(vw[2][w], vw[3][w], 0x7632);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816<C>(o[nt][w], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                }
            }
        }
        cp_async_wait<0>();

        // ---- the warps' rows together -------------------------------------------------------------------------------
        const float unit = C == kBf16 ? 1.f : exp2_fast((C == kE4m3 && vexp != -200 ? (float)vexp : 0.f) - kShift);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float sum = l[nt][c];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int row = nt * 8 + 2 * t + c;
                if (g == 0) { sm.m[warp][row] = m[nt][c]; sm.l[warp][row] = sum; }
                // values 2k and 2k+1 of this lane's D/8
#pragma unroll
                for (int k = 0; k < Sh::kMTiles; k += 2)
                    *reinterpret_cast<float4*>(rows_of(warp) + row * D + g * (D / 8) + 2 * k) =
                        make_float4(o[nt][k][c] * unit, o[nt][k][c + 2] * unit, o[nt][k + 1][c] * unit, o[nt][k + 1][c + 2] * unit);
            }
        __syncthreads();
        if (tid < R) {
            float top = -inf, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) top = fmaxf(top, sm.m[w][tid]);
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) {
                const float f = sm.m[w][tid] == -inf ? 0.f : exp2_fast(sm.m[w][tid] - top);
                sm.weight[w][tid] = f;
                sum += sm.m[w][tid] == -inf ? sm.l[w][tid] : f * sm.l[w][tid];  // (a NaN sum stays one)
            }
            sm.row_m[tid] = top;
            sm.row_l[tid] = sum;
        }
        __syncthreads();
        const unsigned long long item_last = item_first + s.units - 1;
        const int c0 = (int)(((item_first + 1) * n_cta - 1) / total), c1 = (int)(((item_last + 1) * n_cta - 1) / total);
        const bool whole = c0 == c1;
        constexpr int kRowFloats = D + 2;
        float* part = p.partial + ((int64_t)blockIdx.x * 2 + ((int)blockIdx.x == c0 ? 1 : 0)) * kAttnMaxRows * kRowFloats;
        auto write_row = [&](int row, int d, const float4 v, float sum, float top) {
            const int r = row0 + row;
            const int64_t tok = s.r.q0 + r / p.G;
            const int head = s.h * p.G + r % p.G;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            uint2 w;
            if constexpr (kQBf16) {
                w.x = pack_p<kBf16>(v.x * inv, v.y * inv);
                w.y = pack_p<kBf16>(v.z * inv, v.w * inv);
            } else {
                w.x = pack_p<kF16>(v.x * inv, v.y * inv);
                w.y = pack_p<kF16>(v.z * inv, v.w * inv);
            }
            *reinterpret_cast<uint2*>(static_cast<QT*>(p.out) + tok * p.os_t + (int64_t)head * p.os_h + d) = w;
            if (d == 0 && p.lse != nullptr) p.lse[tok * p.Hq + head] = sum == 0.f ? -inf : (top + log2f(sum)) * 0.69314718055994531f;
        };
        for (int i = tid; i < R * D / 4; i += kDecWarps * 32) {
            const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
            if (row0 + row >= n_rows) continue;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) {
                if (sm.m[w][row] == -inf) continue;
                const float f = sm.weight[w][row];
                const float4 x = *reinterpret_cast<const float4*>(rows_of(w) + row * D + d);
                v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
            }
            if (whole) {
                write_row(row, d, v, sm.row_l[row], sm.row_m[row]);
            } else {
                *reinterpret_cast<float4*>(part + row * D + d) = v;
                if (d == 0) {
                    part[kAttnMaxRows * D + row] = sm.row_m[row];
                    part[kAttnMaxRows * (D + 1) + row] = sm.row_l[row];
                }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int old = atom_add_release_gpu(p.counters + c0, 1);
                sm.last = old == c1 - c0;
                if (sm.last) p.counters[c0] = 0;
            }
            __syncthreads();
            if (sm.last) {
                __threadfence();
                attn_join<D, kAttnMaxRows, kDecWarps, QT>(p, c0, c1, s.r.q0, s.h, row0, min(R, n_rows - row0), warp, lane);
            }
        }
        __syncthreads();  // the shared rows are used again
        u = item_first + s.last;
    }
}

template <int D, int C, int NT, typename QT>
static int launch_decode(const AttnParams& p, cudaStream_t st)
{
    // stages: as many 16-token tiles per warp as two resident CTAs have room for
    constexpr int kFit = (112 * 1024 - 4096) / (DecShape<D, C>::kStage * kDecWarps);
    constexpr int STAGES = kFit < 2 ? 2 : kFit > 6 ? 6 : kFit;
    constexpr size_t smem = sizeof(DecShared<D, C, NT, STAGES>);
    static_assert(smem <= 227 * 1024, "shared memory");
    auto kernel = decode_kernel<D, C, NT, STAGES, QT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) { note_cuda_error(e); (void)cudaGetLastError(); return UCMR_ERR_LAUNCH; }
    int resident = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kDecWarps * 32, smem);
    if (e != cudaSuccess) { note_cuda_error(e); (void)cudaGetLastError(); return UCMR_ERR_LAUNCH; }
    int ctas = device_sms() * (resident < 1 ? 1 : resident);
    if (ctas > kAttnMaxCtas) ctas = kAttnMaxCtas;
    return launch_kernel(kernel, dim3(ctas), dim3(kDecWarps * 32), smem, st, p);
}

template <int D, int C, typename QT>
static int launch_rows(const AttnParams& p, int64_t rows, cudaStream_t st)
{
    // up to eight rows fill one column group; more take two, so that the keys are read once for 16 rows
    return rows <= 8 ? launch_decode<D, C, 1, QT>(p, st) : launch_decode<D, C, 2, QT>(p, st);
}

template <int D>
static int launch_types(const AttnParams& p, int dtype, int cache_dtype, int64_t rows, cudaStream_t st)
{
    if (cache_dtype == UCMR_E4M3)
        return dtype == UCMR_BF16 ? launch_rows<D, kE4m3, __nv_bfloat16>(p, rows, st) : launch_rows<D, kE4m3, __half>(p, rows, st);
    return dtype == UCMR_BF16 ? launch_rows<D, kBf16, __nv_bfloat16>(p, rows, st) : launch_rows<D, kF16, __half>(p, rows, st);
}

}  // namespace ucmr

extern "C" size_t ucmr_paged_attention_workspace_bytes(int head_dim)
{
    return head_dim > 0 ? ucmr::attn_workspace_bytes(head_dim) : 0;
}

extern "C" int ucmr_paged_attention_workspace_init(void* workspace, size_t bytes, void* stream)
{
    constexpr size_t head = UCMR_WORKSPACE_HEADER_BYTES + ucmr::kAttnCounterBytes;
    if (!workspace || bytes < head) return UCMR_ERR_WORKSPACE;
    cudaError_t e = cudaMemsetAsync(workspace, 0, head, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) { ucmr::note_cuda_error(e); (void)cudaGetLastError(); return UCMR_ERR_LAUNCH; }
    return UCMR_OK;
}

extern "C" int ucmr_paged_attention(const void* q, int64_t T, int Hq, int D, int64_t q_stride_t, int64_t q_stride_h, int dtype,
                                    const void* k_cache, int64_t kc_stride_block, int64_t kc_stride_t, int64_t kc_stride_h,
                                    const void* v_cache, int64_t vc_stride_block, int64_t vc_stride_t, int64_t vc_stride_h,
                                    int64_t NB, int BS, int Hkv, int cache_dtype, const float* k_scale, const float* v_scale,
                                    const int32_t* block_table, int max_blocks, int64_t bt_stride_b, int64_t bt_stride_h,
                                    const int32_t* seq_lens, const int32_t* query_start, int max_query_len, int B, float scale,
                                    int causal, void* out, int64_t o_stride_t, int64_t o_stride_h, float* lse, void* workspace,
                                    size_t workspace_bytes, void* stream)
{
    using namespace ucmr;
    if (T < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || NB < 0 || BS <= 0 || B < 0 || max_blocks < 0 || max_query_len < 0)
        return UCMR_ERR_BAD_ARG;
    if (!query_start && T != B) return UCMR_ERR_BAD_ARG;
    if (dtype != UCMR_BF16 && dtype != UCMR_FP16) return UCMR_ERR_UNSUPPORTED;
    if (cache_dtype != dtype && cache_dtype != UCMR_E4M3) return UCMR_ERR_UNSUPPORTED;
    if (cache_dtype == UCMR_E4M3 ? (!k_scale || !v_scale) : (k_scale || v_scale)) return UCMR_ERR_BAD_ARG;
    if (D != 64 && D != 128) return UCMR_ERR_UNSUPPORTED;
    if (T > 0x7FFFFFFF || NB > 0x7FFFFFFF || (int64_t)max_blocks * BS > 0x7FFFFF00 || (int64_t)max_query_len * (Hq / Hkv) > 0x7FFFFFFF)
        return UCMR_ERR_UNSUPPORTED;
    if (B == 0 || T == 0) return UCMR_OK;
    if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out) return UCMR_ERR_BAD_ARG;
    if (!workspace || workspace_bytes < attn_workspace_bytes(D)) return UCMR_ERR_WORKSPACE;
    const int es = cache_dtype == UCMR_E4M3 ? 1 : 2;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(workspace);
    const int64_t cs = (kc_stride_block | kc_stride_t | kc_stride_h | vc_stride_block | vc_stride_t | vc_stride_h) * es;
    const uintptr_t qo = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out);
    const int64_t qs = q_stride_t | q_stride_h | o_stride_t | o_stride_h;
    if (bits % 16 != 0 || cs % 16 != 0 || qo % 16 != 0 || qs % 8 != 0) return UCMR_ERR_UNSUPPORTED;

    AttnParams p{};
    p.q = q; p.qs_t = q_stride_t; p.qs_h = q_stride_h;
    p.cache[0] = k_cache; p.cs_b[0] = kc_stride_block * es; p.cs_t[0] = kc_stride_t * es; p.cs_h[0] = kc_stride_h * es;
    p.cache[1] = v_cache; p.cs_b[1] = vc_stride_block * es; p.cs_t[1] = vc_stride_t * es; p.cs_h[1] = vc_stride_h * es;
    p.scale[0] = k_scale; p.scale[1] = v_scale;
    p.NB = NB; p.BS = BS; p.Hkv = Hkv; p.Hq = Hq; p.G = Hq / Hkv; p.by_block = FastDiv::by((uint32_t)BS);
    p.table = block_table; p.bt_b = bt_stride_b; p.bt_h = bt_stride_h; p.max_blocks = max_blocks;
    p.seq_lens = seq_lens; p.query_start = query_start; p.T = T; p.B = B;
    p.scale_log2 = scale * 1.4426950408889634f; p.causal = causal;
    p.out = out; p.os_t = o_stride_t; p.os_h = o_stride_h; p.lse = lse;
    p.status = static_cast<int32_t*>(workspace);
    p.counters = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + UCMR_WORKSPACE_HEADER_BYTES);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + UCMR_WORKSPACE_HEADER_BYTES + kAttnCounterBytes);
    const int64_t rows = (int64_t)(query_start ? max_query_len : 1) * p.G;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows > 16) return attention_tiles(p, D, dtype, cache_dtype, st);
    switch (D) {
        case 64: return launch_types<64>(p, dtype, cache_dtype, rows, st);
        default: return launch_types<128>(p, dtype, cache_dtype, rows, st);
    }
}
