// Attention over the paged KV cache (sm_100a): out = softmax(scale * q k^T) v over the tokens of the blocks that a table
// lists, for up to 16 rows per (request, kv head): decode steps and short verifications.  Calls with more rows go to
// paged_prefill.cu (verification of 4 tokens with 8 query heads per kv head, 32 rows: 112 us there, 205 us here in two row
// tiles; 16 rows, 16 requests of 8192 tokens: 128 us here, 139 us there).  Cache of 16-bit values, or of e4m3 codes with a scale
// per (block, kv head).
//
// Work.  The G query heads of a kv head times the request's query tokens are rows; 4, 8 or 16 of them (a row tile) share one
// pass over the keys.  An item is (request, row tile, up to four kv heads side by side); its tokens are cut into units.  All
// units of all items form one line, which is divided evenly over the CTAs (two per SM where registers and shared memory
// allow it): ragged batches balance, and one long request is split over the whole GPU.  A CTA that has only a part of an item
// leaves (max, sum, unnormalised rows) in its slot of the workspace; the last of an item's CTAs to arrive adds the parts up,
// in the order of the tokens: results do not depend on timing.
//
// Eight warps, each with one of the item's heads and every n-th group of 16 tokens; they do not wait for one another until
// the item ends.  Each has a ring of stages of 16 tokens in shared memory.  Where a block holds a multiple of 16 tokens, one
// thread has the copy engine fetch a stage's keys and values (boxes of 16 tokens of a head; a mbarrier tells when they are
// there): 16 x 131072 tokens 952 -> 735 us in short runs against copies by all lanes, which were bound by their instructions.  Otherwise all
// lanes copy, 16 bytes at a time, with block ids and tails per token: any block size, any strides.
//   S^T = K Q^T: tokens are the 16 rows of the matrix instruction, query rows its 8 columns.  The order in which the products
//     run over the head dimension is free, so each lane takes 16 consecutive bytes of a key (4 lanes per key), and the
//     queries are read in the same order.
//   O^T += V^T P^T: the head dimension is the 16 rows, again in a free order: each lane takes D/8 consecutive values of four
//     tokens, and interleaves the tokens two by two for its fragments.  P^T is S^T's fragment, transposed by movmatrix.
// mma.sync serves here because the rows are few: 16 x 8 tiles waste little, where a tile of the tensor memory has 128 rows.
//
// Numerics.  e4m3 codes against bf16 queries: the query row, after a power of two has brought its largest value to 448 or
// less, is the sum of two e4m3 values (4 + 4 of bf16's 8 significant bits): exactly for elements down to 2^-9 of the row's
// largest, and to half of 2^-9, which is 2^-17 of the row's largest, for smaller ones.  So keys are multiplied as the codes
// they are, by two columns per query row, m16n8k32, whose sums are float32.  Against fp16 queries (11 bits) codes become fp16,
// exactly, and so do the queries after a power of two per row.  Scores, softmax and rows are float32; the key scale and the
// softmax scale are applied to the float32 score.  The probability that multiplies V is rounded to fp16 (half a step: 2^-11)
// with the value scale folded in, counted from 2^(14 - E), E the exponent of the largest value scale so far: the largest
// product is 2^14, so probabilities down to 2^-28 of the largest keep all bits and those below 2^-39 are dropped.  (E is -112 at
// least: 2^(14 - E) and 2^(E - 14) are normal numbers.  Before scales of 2^-126 that leaves a largest product of 1.)  A bf16
// cache uses bf16 operands (probabilities rounded by 2^-8), an fp16 cache fp16 ones.
//
// What bounds it: HBM for 16-bit caches (64 x 4096 tokens in bf16, 4 rows: 179 us, 6.0 TB/s); the issue of instructions and
// their latencies for e4m3, so that time goes with the SM clock: 16 x 131072 tokens, 8 heads of 128, 4 rows, take 735 us (5.8
// TB/s) in short runs at 1965 MHz and 850 us (5.05 TB/s) in long ones, where the power limit holds the clock near 1.7 GHz (memory
// clock unchanged); 8 rows 970 us, 16 rows 1350 us.  Calls of some 10 us of traffic pay 20 to 30 us for the launch, the line,
// the first copies and the join (16 x 8192 tokens: 70 us for 268 MB).
#include <cuda.h>

#include "paged_attention.cuh"

namespace ucmr {

int device_sms();
int attention_tiles(const AttnParams& p, int D, int dtype, int cache_dtype, cudaStream_t st);  // paged_prefill.cu

enum { kBf16 = 0, kF16 = 1, kE4m3 = 2 };

constexpr float kShift = 14.f;  // see "Numerics"

// A warp's stage: 16 tokens' keys, then their values, each as 16 rows of 64 or 128 bytes (rows of 256 bytes as two halves),
// with the swizzle of the bulk tensor copies: 16-byte piece c of row r lies at piece c ^ (r % 8), or c ^ (r / 2 % 4).
template <int D, int C>
struct DecShape {
    static constexpr int kEs = C == kE4m3 ? 1 : 2;          // bytes per cached value
    static constexpr int kRow = D * kEs;                    // bytes per key
    static constexpr int kTile = 16 * kRow;
    static constexpr int kStage = 2 * kTile;
    static constexpr int kKPieces = kRow / 64;              // 16-byte pieces of a key per lane
    static constexpr int kVBytes = kRow / 8;                // bytes of a value row per lane
    static constexpr int kKSteps = D / 16;
    static constexpr int kMTiles = D / 16;

    static __device__ __forceinline__ uint32_t at(int row, int piece)
    {
        if constexpr (kRow == 64) return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4);
        return (piece >> 3) * 2048 + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
    }
    // Orders that are free, chosen so that the eight lanes that read together meet no bank twice: the token that lane g holds
    // as row g of the products, and which eighth of a value row it holds.
    static __device__ __forceinline__ int token(int g) { return kRow == 64 ? g : (g & 1) * 4 + (g >> 1); }
    static __device__ __forceinline__ int eighth(int g)
    {
        return kRow == 64 ? g : kRow == 128 ? (g & 1) * 4 + (g >> 1) : (g & 4) | ((g & 1) << 1) | ((g >> 1) & 1);
    }
};


__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// 16 tokens of one head; x in elements, a multiple of 128 bytes
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int x, int head, int row, int block, uint64_t* bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(head), "r"(row), "r"(block), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int C>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (C == kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
    return r;
}

// Two values as e4m3 codes, the first in the low byte; |v| up to 448.  Values that are not finite become NaN.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    if (!(fabsf(lo) <= 3.402823466e38f)) r = (uint16_t)((r & 0xff00u) | 0x7fu);
    if (!(fabsf(hi) <= 3.402823466e38f)) r = (uint16_t)((r & 0xffu) | 0x7f00u);
    return r;
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return reinterpret_cast<const __half2&>(v); }

__device__ __forceinline__ void mma_16832(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// How a CTA's warps share an item: `heads` kv heads side by side times `tokens` groups of 16 tokens.
struct DecPlan {
    int heads, tokens, groups;  // groups: of heads, each an item of its own
    int unit;                   // tokens per unit of the line
    int extra;                  // units that an item counts for its fixed cost
};

// One of the CTA's stretches: units [first, last) of one item.
struct Segment {
    int b, rt, h, first, last, units;
    AttnRequest r;
};

constexpr int kDecWarps = 8;
constexpr int kDecThreads = kDecWarps * 32;

// Residence: two CTAs per SM with up to 128 registers a thread, where the rows (16 of them hold 64 registers) and the stages
// (32 tokens of 256-byte rows take 16 KB) leave room; else one CTA.  As many stages as fit.
template <int D, int C, int NG>
struct DecConfig {
    static constexpr int kCtas = NG > 2 || DecShape<D, C>::kRow > 128 ? 1 : 2;
    static constexpr int kFit = ((kCtas == 2 ? 112 : 224) * 1024 - 10 * 1024) / (kDecWarps * DecShape<D, C>::kStage);
    static constexpr int kStages = kFit > 6 ? 6 : kFit;
    static_assert(kStages >= 2, "shared memory");
};

template <int D, int C, int NG>
struct DecShared {
    static constexpr int NT = (NG + 1) / 2;
    static constexpr int kStages = DecConfig<D, C, NG>::kStages;
    alignas(1024) unsigned char ring[kDecWarps][kStages][DecShape<D, C>::kStage];
    float scale[kDecWarps][kStages][32];          // 16 key scales, 16 value scales
    uint32_t live[kDecWarps][kStages];            // tokens that are there
    alignas(8) uint64_t landed[kDecWarps][kStages];
    // (a warp's rows take the place of its own ring once its copies have landed)
    static_assert(sizeof(ring[0]) >= NT * 8 * D * 4, "rows do not fit the ring");
    static_assert(sizeof(ring) >= kDecWarps * 4 * (D + 1) * 4, "the join's sums do not fit the ring");
    float m[kDecWarps][NT * 8], l[kDecWarps][NT * 8];
    float weight[kDecWarps][NT * 8];
    float row_m[kDecWarps][NT * 8], row_l[kDecWarps][NT * 8];
    unsigned long long sums[kDecWarps];
    unsigned long long start_units;
    int start_b;
    int last;
};

template <int D, int C, int NG, bool TMA, typename QT>
__global__ void __launch_bounds__(kDecThreads, DecConfig<D, C, NG>::kCtas)
    decode_kernel(const __grid_constant__ AttnParams p, const DecPlan plan, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map)
{
    using Sh = DecShape<D, C>;
    using Smem = DecShared<D, C, NG>;
    constexpr int NT = Smem::NT;
    constexpr int STAGES = DecConfig<D, C, NG>::kStages;
    extern __shared__ unsigned char s_raw[];
    Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    constexpr int R = NG * 4, kSlotRows = kDecWarps * R;
    auto rows_of = [&](int w) { return reinterpret_cast<float*>(&sm.ring[w][0][0]); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    constexpr bool kQBf16 = __is_same(QT, __nv_bfloat16);
    constexpr bool kQ8 = C == kE4m3 && kQBf16;  // keys stay codes: see "Numerics"

    if (TMA && tid < kDecWarps * STAGES) mbar_init(&sm.landed[0][0] + tid, 1);
    if (TMA) fence_mbar_init();
    uint32_t phases = 0;                           // of this warp's barriers, a bit per stage

    // ---- this CTA's stretch of the line of units -------------------------------------------------------------
    auto units_of = [&](const AttnRequest& r) { return (r.len + plan.unit - 1) / plan.unit; };
    auto tiles_of = [&](const AttnRequest& r) { return (int)(((int64_t)r.nq * p.G + R - 1) / R); };
    // (an item without tokens still takes one unit: its rows are written as empty)
    auto line_of = [&](int b) -> unsigned long long {
        const AttnRequest r = attn_request(p, b);
        return (unsigned long long)(max(1, units_of(r)) + plan.extra) * (unsigned)tiles_of(r) * (unsigned)plan.groups;
    };
    const int per = (p.B + kDecThreads - 1) / kDecThreads;
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
            const unsigned long long n = (unsigned long long)(s.units + plan.extra) * (unsigned)tiles_of(s.r) * (unsigned)plan.groups;
            if (u < b_first + n) break;
            b_first += n;
            ++b;
        }
        const int length = s.units + plan.extra;      // (units, and what an item costs besides)
        const unsigned long long in_b = u - b_first;
        const int item = (int)(in_b / length);
        s.b = b;
        s.rt = item / plan.groups;
        const int h0 = (item - s.rt * plan.groups) * plan.heads, nh = min(plan.heads, p.Hkv - h0);
        s.first = (int)(in_b - (unsigned long long)item * length);
        const unsigned long long item_first = u - s.first;
        u = item_first + length;
        if (s.first >= s.units) continue;
        s.last = (int)min((unsigned long long)s.units, u1 - item_first);
        const int row0 = s.rt * R, n_rows = s.r.nq * p.G;  // rows of the request; this tile holds [row0, row0 + R)
        const int hl = warp % plan.heads, tg = warp / plan.heads;     // this warp's head and token group
        const bool busy = hl < nh && tg < plan.tokens;
        s.h = h0 + (busy ? hl : 0);

        // ---- queries: fragments of the second operand.  Column n of a group of eight is row (n % 2) * 4 + n / 2, so that a
        // lane's two columns 2t and 2t+1 are rows t and t + 4; with codes for both operands the columns 2j and 2j+1 of a group
        // of four rows are the two pieces of row j.
        constexpr int kQRegs = kQ8 ? NG : NT, kQSteps = kQ8 ? D / 32 : Sh::kKSteps;
        uint32_t qf[kQRegs][kQSteps][2];
        float qmul[NT][2];  // score factor of the lane's columns
        int limit[NT][2];
        int max_limit = 0, min_limit = 0x7fffffff;
        float mul[kQRegs];
#pragma unroll
        for (int nt = 0; nt < kQRegs; ++nt) {
            const int in_tile = kQ8 ? nt * 4 + (g >> 1) : nt * 8 + (g & 1) * 4 + (g >> 1), row = row0 + in_tile;
            const bool live = row < n_rows && in_tile < R;
            const QT* qr = static_cast<const QT*>(p.q);
            if (live) qr += (int64_t)(s.r.q0 + row / p.G) * p.qs_t + (int64_t)(s.h * p.G + row % p.G) * p.qs_h;
            // A lane's elements come in the order in which it holds a key's bytes: 16 consecutive bytes of every 64.
            constexpr int kVec = kQ8 ? 8 : 4;    // elements per step and lane
            uint32_t raw[kQSteps][kVec / 2];
#pragma unroll
            for (int ks = 0; ks < kQSteps; ++ks) {
                constexpr int kPerPiece = 16 / Sh::kEs / kVec;
                const int d = (ks / kPerPiece) * (64 / Sh::kEs) + t * (16 / Sh::kEs) + (ks % kPerPiece) * kVec;
#pragma unroll
                for (int i = 0; i < kVec / 2; ++i) raw[ks][i] = 0;
                if (live) {
                    if constexpr (kQ8) {
                        const uint4 v = *reinterpret_cast<const uint4*>(qr + d);
                        raw[ks][0] = v.x; raw[ks][1] = v.y; raw[ks][2] = v.z; raw[ks][kVec / 2 - 1] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(qr + d);
                        raw[ks][0] = v.x; raw[ks][1] = v.y;
                    }
                }
            }
            mul[nt] = 1.f;
            if constexpr (C == kE4m3) {
                uint32_t big = 0;  // largest finite magnitude of the row, as float bits
#pragma unroll
                for (int ks = 0; ks < kQSteps; ++ks)
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        const uint32_t v = __float_as_uint(fabsf(unpack_16(raw[ks][i >> 1], i & 1, kQBf16)));
                        if (v < 0x7f800000u) big = max(big, v);
                    }
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                // 2^e <= big < 2^(e+1).  fp16: the row times 2^-e lies below 2.  Codes: up to 448 = 1.75 * 2^8.
                int e = big == 0 ? 0 : max(-110, min(120, (int)(big >> 23) - 127));
                if (kQ8) e -= (big & 0x7fffffu) > 0x600000u ? 7 : 8;
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                mul[nt] = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int ks = 0; ks < kQSteps; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if constexpr (kQ8) {
                            float v[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) v[j] = unpack_16(raw[ks][2 * i + (j >> 1)], j & 1, true) * down;
                            const uint32_t lo2 = to_e4m3x2(v[0], v[1]), hi2 = to_e4m3x2(v[2], v[3]);
                            uint32_t code = lo2 | (hi2 << 16);
                            if (g & 1) {                 // the second piece: what the first leaves
                                const float2 a = __half22float2(as_half2(e4m3x2_to_f16x2(lo2))), b2 = __half22float2(as_half2(e4m3x2_to_f16x2(hi2)));
                                code = to_e4m3x2(v[0] - a.x, v[1] - a.y) | (to_e4m3x2(v[2] - b2.x, v[3] - b2.y) << 16);
                            }
                            qf[nt][ks][i] = code;
                        } else {
                            qf[nt][ks][i] = pack_p<kF16>(unpack_16(raw[ks][i], 0, kQBf16) * down, unpack_16(raw[ks][i], 1, kQBf16) * down);
                        }
                    }
            } else {
#pragma unroll
                for (int ks = 0; ks < kQSteps; ++ks) { qf[nt][ks][0] = raw[ks][0]; qf[nt][ks][1] = raw[ks][1]; }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float of = kQ8 ? mul[nt * 2 + i < kQRegs ? nt * 2 + i : 0] : mul[nt < kQRegs ? nt : 0];
                qmul[nt][i] = __shfl_sync(0xffffffffu, of, kQ8 ? 8 * t : 8 * t + 4 * i) * p.scale_log2;
                const int in_tile = nt * 8 + t + 4 * i, r2 = row0 + in_tile;
                limit[nt][i] = r2 < n_rows && in_tile < R ? attn_limit(p, s.r, r2 / p.G) : 0;
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
        float vup = 0.f;  // 2^(14 - E)
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
        const int mine = Sh::token(g);                 // token (and that + 8) whose scores this lane has
        // this warp's 16 tokens out of every plan.tokens * 16
        const int seg_tok = s.first * plan.unit, seg_end = min(s.last * plan.unit, max_limit);
        const int stride = plan.tokens * 16, from_tok = seg_tok + tg * 16;
        const int n_tiles = busy && from_tok < seg_end ? (seg_end - from_tok + stride - 1) / stride : 0;
        auto tok_at = [&](int i) { return from_tok + i * stride; };
        auto block_of = [&](int i) {
            const int tok = tok_at(i) + (lane & 15);
            return i < n_tiles && tok < max_limit ? table[p.by_block.div(tok)] : -1;
        };
        // Any block size and strides: block ids, rows and tails token by token, 16-byte asynchronous copies.
        auto issue_rows = [&](int st, int tok16, int blk) {   // lanes 0-15 and 16-31: the blocks of the 16 tokens
            const int tok = tok16 + (lane & 15);
            const bool in = tok < max_limit;
            const bool live = in && blk >= 0 && blk < p.NB;
            if (in && !live) flag_status(p.status, UCMR_DEV_BAD_BLOCK_ID);
            const int row = tok - p.by_block.div(tok) * p.BS;
            const uint32_t mask = __ballot_sync(0xffffffffu, live) & 0xffffu;
#pragma unroll
            for (int kind = 0; kind < 2; ++kind) {
                const int64_t off = live ? blk * p.cs_b[kind] + row * p.cs_t[kind] + s.h * p.cs_h[kind] : 0;
                const char* base = static_cast<const char*>(p.cache[kind]);
#pragma unroll
                for (int j = 0; j < Sh::kTile / 512; ++j) {
                    constexpr int kPer = Sh::kRow / 16;
                    const int r = (j * 32 + lane) / kPer, piece = (j * 32 + lane) % kPer;
                    const char* src = base + __shfl_sync(0xffffffffu, off, r) + piece * 16;
                    const bool on = (mask >> r) & 1u;
                    cp_async16(ring + st * Sh::kStage + kind * Sh::kTile + Sh::at(r, piece), on ? src : base, on);
                }
            }
            if constexpr (C == kE4m3) {
                const float* sc = p.scale[lane >> 4];
                cp_async4(smem_u32(&sm.scale[warp][st][lane]), live ? sc + (int64_t)blk * p.Hkv + s.h : sc, live);
            }
            if (lane == 0) sm.live[warp][st] = mask;
        };
        // Block sizes that are multiples of 16: 16 tokens lie in one block side by side, and one thread has the copy engine
        // fetch them (rows behind a length are there, and are not looked at).
        auto issue_tile = [&](int st, int tok16, int blk) {
            const bool there = (unsigned)blk < (unsigned)p.NB;
            if (lane == 0) {
                if (there) {
                    const int row = tok16 - p.by_block.div(tok16) * p.BS;
                    uint64_t* bar = &sm.landed[warp][st];
                    mbar_expect_tx(bar, Sh::kStage);
                    const uint32_t to = ring + st * Sh::kStage;
#pragma unroll
                    for (int x = 0; x < Sh::kRow; x += 128) {
                        load_tile(to + x * 16, &k_map, x / Sh::kEs, s.h, row, blk, bar);
                        load_tile(to + Sh::kTile + x * 16, &v_map, x / Sh::kEs, s.h, row, blk, bar);
                    }
                } else {
                    flag_status(p.status, UCMR_DEV_BAD_BLOCK_ID);
                }
                const int n = min(16, max_limit - tok16);
                sm.live[warp][st] = there ? (1u << n) - 1 : 0u;
            }
            if constexpr (C == kE4m3)
                if (there && lane < 2) cp_async4(smem_u32(&sm.scale[warp][st][lane * 16]), p.scale[lane] + (int64_t)blk * p.Hkv + s.h);
        };
        auto issue = [&](int i, int blk) {
            if constexpr (TMA) issue_tile(i % STAGES, tok_at(i), __shfl_sync(0xffffffffu, blk, 0));
            else issue_rows(i % STAGES, tok_at(i), blk);
        };

        int next = block_of(0);
#pragma unroll 1
        for (int i = 0; i < STAGES - 1; ++i) {
            const int blk = next;
            next = block_of(i + 1);
            if (i < n_tiles) issue(i, blk);
            cp_async_commit();
        }
#pragma unroll 1
        for (int i = 0; i < n_tiles; ++i) {
            {
                const int blk = next;
                next = block_of(i + STAGES);
                __syncwarp();  // every lane is done with the stage that is filled now
                if (i + STAGES - 1 < n_tiles) issue(i + STAGES - 1, blk);
                cp_async_commit();
            }
            cp_async_wait<STAGES - 1>();
            __syncwarp();  // scales and marks come from other lanes
            const int slot = i % STAGES;
            uint32_t mark = sm.live[warp][slot];
            if ((mark & 0xffffu) == 0) continue;
            if constexpr (TMA) {
                if (!mbar_wait(&sm.landed[warp][slot], (phases >> slot) & 1)) {
                    flag_status(p.status, UCMR_DEV_WAIT_TIMEOUT);
                    mark = 0;
                }
                phases ^= 1u << slot;
            }
            const unsigned char* st = &sm.ring[warp][slot][0];
            const bool whole = (mark & 0xffffu) == 0xffffu;
            const int tok0 = tok_at(i);

            // scores of the tokens token(g) and token(g) + 8
            float sc[kQRegs][4];
#pragma unroll
            for (int nt = 0; nt < kQRegs; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
            for (int c = 0; c < Sh::kKPieces; ++c) {
                uint32_t wl[4], wh[4];
                const uint4 lo = *reinterpret_cast<const uint4*>(st + Sh::at(mine, c * 4 + t));
                const uint4 hi = *reinterpret_cast<const uint4*>(st + Sh::at(mine + 8, c * 4 + t));
                wl[0] = lo.x; wl[1] = lo.y; wl[2] = lo.z; wl[3] = lo.w;
                wh[0] = hi.x; wh[1] = hi.y; wh[2] = hi.z; wh[3] = hi.w;
                if constexpr (kQ8) {
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int nt = 0; nt < kQRegs; ++nt)
                            mma_16832(sc[nt], wl[2 * w], wh[2 * w], wl[2 * w + 1], wh[2 * w + 1],
                                      qf[nt][c * 2 + w][0], qf[nt][c * 2 + w][1]);
                } else if constexpr (C == kE4m3) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = e4m3x2_to_f16x2(wl[w]), a2 = e4m3x2_to_f16x2(wl[w] >> 16);
                        const uint32_t a1 = e4m3x2_to_f16x2(wh[w]), a3 = e4m3x2_to_f16x2(wh[w] >> 16);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_16816<C>(sc[nt], a0, a1, a2, a3, qf[nt][c * 4 + w][0], qf[nt][c * 4 + w][1]);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_16816<C>(sc[nt], wl[2 * w], wh[2 * w], wl[2 * w + 1], wh[2 * w + 1],
                                         qf[nt][c * 2 + w][0], qf[nt][c * 2 + w][1]);
                }
            }
            float vfac[2], kfac[2];
            float vdown = 1.f;
            if constexpr (C == kE4m3) {
                uint32_t big = 0;
                const float* f = sm.scale[warp][slot];
                const int one = TMA ? 0 : mine, two = TMA ? 0 : mine + 8;    // (one scale for all 16 tokens of a block)
                kfac[0] = f[one]; kfac[1] = f[two];
                vfac[0] = f[16 + one]; vfac[1] = f[16 + two];
                big = max(big, max(__float_as_uint(fabsf(vfac[0])), __float_as_uint(fabsf(vfac[1]))));
                if (!TMA) big = __reduce_max_sync(0xffffffffu, big);   // (the same in all lanes otherwise)
                const int e = max(-112, min(128, (int)(big >> 23) - 126));  // every scale is below 2^e
                if (e > vexp) {
                    vdown = vexp == -200 ? 0.f : exp2_fast((float)(vexp - e));
                    vexp = e;
                    vup = exp2_fast(kShift - (float)vexp);  // a power of two
                }
                vfac[0] *= vup; vfac[1] *= vup;
            } else {
                vfac[0] = vfac[1] = C == kBf16 ? 1.f : 16384.f; kfac[0] = kfac[1] = 1.f;
            }
            const bool edge = !whole || tok0 + 16 > min_limit;
            bool grown = vdown != 1.f;
            float alpha[NT][2];
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                constexpr int kLast = NG - 2 * (NT - 1);     // rows t and, but for the last of an odd number of fours, t + 4
                const int cols = nt == NT - 1 ? kLast : 2;
                float x[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    x[c] = 0.f;
                    if ((c & 1) >= cols) continue;
                    float v;
                    if constexpr (kQ8) {
                        const int group = nt * 2 + (c & 1) < kQRegs ? nt * 2 + (c & 1) : 0;
                        v = sc[group][c & 2] + sc[group][(c & 2) + 1];
                    } else {
                        v = sc[nt < kQRegs ? nt : 0][c];
                    }
                    x[c] = v * (kfac[c >> 1] * qmul[nt][c & 1]);
                    if (edge) {
                        const int tk = mine + 8 * (c >> 1);
                        if (!((mark >> tk) & 1u) || tok0 + tk >= limit[nt][c & 1]) x[c] = -inf;
                    }
                }
                float top[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) top[c] = fmaxf(x[c], x[c + 2]);
#pragma unroll
                for (int w = 4; w < 32; w <<= 1)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        if (c < cols) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], w));
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    alpha[nt][c] = 1.f;
                    if (c >= cols) continue;
                    if (top[c] > m[nt][c]) {
                        alpha[nt][c] = exp2_fast(m[nt][c] - top[c]);  // (0 from -inf)
                        m[nt][c] = top[c];
                        grown = true;
                    }
                    const float ref = m[nt][c] == -inf ? 0.f : m[nt][c];
                    const float p0 = exp2_fast(x[c] - ref), p1 = exp2_fast(x[c + 2] - ref);
                    x[c] = p0 * vfac[0];
                    x[c + 2] = p1 * vfac[1];
                    l[nt][c] = l[nt][c] * alpha[nt][c] + (p0 + p1);
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
            // values: D/8 consecutive ones of the tokens that are rows 2t, 2t+1, 2t+8, 2t+9 of the products
            constexpr int W = Sh::kVBytes / 4;
            const unsigned char* sv = st + Sh::kTile;
            const int part = Sh::eighth(g);
            auto value_at = [&](int tk) { return sv + Sh::at(tk, part * Sh::kVBytes / 16) + (part * Sh::kVBytes) % 16; };
            uint32_t vw[4][W];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int tk = Sh::token(2 * t + (k & 1)) + 8 * (k >> 1);
                if constexpr (Sh::kVBytes >= 16) {
#pragma unroll
                    for (int c = 0; c < Sh::kVBytes / 16; ++c) {
                        const uint4 v = *reinterpret_cast<const uint4*>(sv + Sh::at(tk, part * (Sh::kVBytes / 16) + c));
                        vw[k][c * 4] = v.x; vw[k][c * 4 + 1] = v.y; vw[k][c * 4 + 2] = v.z; vw[k][c * 4 + 3] = v.w;
                    }
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(value_at(tk));
                    vw[k][0] = v.x;
                    vw[k][1] = v.y;
                }
            }
            if (edge) {
                // Some rows, or all, do not see some of these tokens: a value that is not finite must not reach them as
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
                        if (!((mark >> tk) & 1u)) continue;
#pragma unroll
                        for (int d = 0; d < D / 8; ++d) {
                            const int byte = d * Sh::kEs;
                            const unsigned char* at;
                            if constexpr (Sh::kVBytes >= 16) at = sv + Sh::at(tk, part * (Sh::kVBytes / 16) + byte / 16) + byte % 16;
                            else at = value_at(tk) + byte;
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
                                    if (tok0 + tk < limit[nt][c]) o[nt][d / 2][(d & 1) * 2 + c] += v;
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
        // (a warp without tokens leaves -inf and zeros)
        const float unit = C == kBf16 ? 1.f : exp2_fast((C == kE4m3 && vexp != -200 ? (float)vexp : 0.f) - kShift);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float sum = l[nt][c];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int row = nt * 8 + t + 4 * c;
                if (row >= R) continue;
                if (g == 0) { sm.m[warp][row] = m[nt][c]; sm.l[warp][row] = sum; }
                // values 2k and 2k+1 of this lane's D/8
#pragma unroll
                for (int k = 0; k < Sh::kMTiles; k += 2)
                    *reinterpret_cast<float4*>(rows_of(warp) + row * D + Sh::eighth(g) * (D / 8) + 2 * k) =
                        make_float4(o[nt][k][c] * unit, o[nt][k][c + 2] * unit, o[nt][k + 1][c] * unit, o[nt][k + 1][c + 2] * unit);
            }
        __syncthreads();
        // the token groups' rows of each head together
        if (tid < kSlotRows) {
            const int h = tid / R, row = tid - h * R;
            if (h < nh) {
                float top = -inf, sum = 0.f;
                for (int w = h; w < plan.heads * plan.tokens; w += plan.heads) top = fmaxf(top, sm.m[w][row]);
                for (int w = h; w < plan.heads * plan.tokens; w += plan.heads) {
                    const float f = sm.m[w][row] == -inf ? 0.f : exp2_fast(sm.m[w][row] - top);
                    sm.weight[w][row] = f;
                    sum += sm.m[w][row] == -inf ? sm.l[w][row] : f * sm.l[w][row];  // (a NaN sum stays one)
                }
                sm.row_m[h][row] = top;
                sm.row_l[h][row] = sum;
            }
        }
        __syncthreads();
        const unsigned long long item_last = item_first + s.units - 1;
        const int c0 = (int)(((item_first + 1) * n_cta - 1) / total), c1 = (int)(((item_last + 1) * n_cta - 1) / total);
        const bool whole_item = c0 == c1;
        constexpr int kRowFloats = D + 2;
        float* part = p.partial + ((int64_t)blockIdx.x * 2 + ((int)blockIdx.x == c0 ? 1 : 0)) * kSlotRows * kRowFloats;
        for (int i = tid; i < nh * R * (D / 4); i += kDecThreads) {
            const int slot_row = i / (D / 4), d = (i - slot_row * (D / 4)) * 4;
            const int h = slot_row / R, row = slot_row - h * R, r = row0 + row;
            if (r >= n_rows) continue;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = h; w < plan.heads * plan.tokens; w += plan.heads) {
                const float f = sm.weight[w][row];
                if (sm.m[w][row] == -inf) continue;
                const float4 x = *reinterpret_cast<const float4*>(rows_of(w) + row * D + d);
                v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
            }
            const float sum = sm.row_l[h][row], top = sm.row_m[h][row];
            if (whole_item) {
                const int64_t tok = s.r.q0 + r / p.G;
                const int head = (h0 + h) * p.G + r % p.G;
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                *reinterpret_cast<uint2*>(static_cast<QT*>(p.out) + tok * p.os_t + (int64_t)head * p.os_h + d) =
                    make_uint2(Out16<QT>::pack(v.x * inv, v.y * inv), Out16<QT>::pack(v.z * inv, v.w * inv));
                if (d == 0 && p.lse != nullptr) p.lse[tok * p.Hq + head] = sum == 0.f ? -inf : (top + log2f(sum)) * 0.69314718055994531f;
            } else {
                *reinterpret_cast<float4*>(part + slot_row * D + d) = v;
                if (d == 0) {
                    part[kSlotRows * D + slot_row] = top;
                    part[kSlotRows * (D + 1) + slot_row] = sum;
                }
            }
        }
        if (!whole_item) {
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
                attn_join<D, kSlotRows, kDecWarps, true, QT>(p, c0, c1, nh * R, warp, lane, rows_of(0), [&](int slot_row, int64_t& tok, int& head) {
                    const int h = slot_row / R, r = row0 + slot_row - h * R;
                    tok = s.r.q0 + r / p.G;
                    head = (h0 + h) * p.G + r % p.G;
                    return r < n_rows;
                });
            }
        }
        if (TMA) fence_proxy_async();  // (plain writes to the ring come before the next copies into it)
        __syncthreads();               // the shared rows are used again
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Maps {D, Hkv, BS, NB} of the two caches for boxes of 16 tokens of a head; false where a map cannot hold the strides.
template <int D, int C>
static bool cache_maps(const AttnParams& p, CUtensorMap (&maps)[2])
{
    static EncodeTiled encode = nullptr;  // resolving twice is harmless
    if (!encode) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) != cudaSuccess) { (void)cudaGetLastError(); return false; }
        if (found != cudaDriverEntryPointSuccess || !ptr) return false;
        encode = reinterpret_cast<EncodeTiled>(ptr);
    }
    constexpr int kEs = DecShape<D, C>::kEs, kRow = DecShape<D, C>::kRow;
    for (int k = 0; k < 2; ++k) {
        if (p.cs_b[k] < 0 || p.cs_t[k] < 0 || p.cs_h[k] < 0) return false;
        const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)p.Hkv, (cuuint64_t)p.BS, (cuuint64_t)p.NB};
        const cuuint64_t strides[3] = {(cuuint64_t)p.cs_h[k], (cuuint64_t)p.cs_t[k], (cuuint64_t)p.cs_b[k]};
        const cuuint32_t box[4] = {(cuuint32_t)((kRow < 128 ? kRow : 128) / kEs), 1, 16, 1}, step[4] = {1, 1, 1, 1};
        const CUtensorMapDataType type = C == kE4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;  // (bits are bits)
        if (encode(&maps[k], type, 4, const_cast<void*>(p.cache[k]), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   kRow < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    }
    return true;
}

template <int D, int C, int NG, typename QT>
static int launch_decode(const AttnParams& p, cudaStream_t st)
{
    constexpr size_t smem = sizeof(DecShared<D, C, NG>) + 1024;
    static_assert(smem <= 227 * 1024 / DecConfig<D, C, NG>::kCtas, "shared memory");
    static_assert((size_t)DecConfig<D, C, NG>::kCtas * kAttnMaxSms * 2 * kDecWarps * NG * 4 <= kAttnPartRows, "workspace");
    CUtensorMap maps[2] = {};
    const bool tiles = p.BS % 16 == 0 && cache_maps<D, C>(p, maps);
    auto kernel = tiles ? decode_kernel<D, C, NG, true, QT> : decode_kernel<D, C, NG, false, QT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) { note_cuda_error(e); (void)cudaGetLastError(); return UCMR_ERR_LAUNCH; }
    const int sms = device_sms(), ctas = (sms < kAttnMaxSms ? sms : kAttnMaxSms) * DecConfig<D, C, NG>::kCtas;
    DecPlan plan;
    // Heads side by side in a CTA: a token's heads lie side by side in memory, but the part that a CTA leaves of an item has
    // the rows of all its heads, and one CTA adds up an item's parts.  So as many heads, up to four, as leave an item about
    // ten parts or fewer.  Measured for 8 heads of 128, e4m3, four rows each, in us with 4 | 2 | 1 heads side by side:
    // 1 request of 131072 tokens 94 | 77 | 68, 4 of 32768 72 | 69 | 72, 16 of 8192 68 | 72 | 74, 200 of 4096 308 | 316 | 341.
    int heads = 4;
    while (heads > 1 && (int64_t)ctas * heads > (int64_t)10 * p.B * p.Hkv) heads /= 2;
    plan.groups = (p.Hkv + heads - 1) / heads;
    plan.heads = (p.Hkv + plan.groups - 1) / plan.groups;
    plan.tokens = kDecWarps / plan.heads;
    // Units of 128 tokens; fewer when even the longest possible batch would not give every CTA two of them.
    plan.unit = 128;
    const int64_t most = (int64_t)p.max_blocks * p.BS;
    if ((most + 127) / 128 * p.B * plan.groups < 2 * ctas) plan.unit = plan.tokens * 16 > 32 ? plan.tokens * 16 : 32;
    plan.extra = 1;
    return launch_kernel(kernel, dim3(ctas), dim3(kDecThreads), smem, st, p, plan, maps[0], maps[1]);
}

template <int D, int C, typename QT>
static int launch_rows(const AttnParams& p, int64_t rows, cudaStream_t st)
{
    // rows in fours: one, two or four of them share a pass over the keys
    if (rows <= 4) return launch_decode<D, C, 1, QT>(p, st);
    return rows <= 8 ? launch_decode<D, C, 2, QT>(p, st) : launch_decode<D, C, 4, QT>(p, st);
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
    if (!q || !k_cache || !v_cache || (!block_table && max_blocks > 0) || !seq_lens || !out) return UCMR_ERR_BAD_ARG;
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
