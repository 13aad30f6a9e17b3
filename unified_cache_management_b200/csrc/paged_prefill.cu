// Attention over the paged KV cache for many rows (sm_100a, tcgen05): prefill chunks, speculative verification, wide
// groups.  Same operator, parameters and numerics as paged_attention.cu, which keeps the calls with up to 16 rows per
// (request, kv head).
//
// One persistent CTA per SM.  The G query heads of a kv head times the request's query tokens are rows; 128 rows are one
// M = 128 tile of the tensor core.  For each tile of 128 tokens: S = Q K^T into TMEM, softmax with one thread per row, P
// back into TMEM as 16-bit values (over the columns of S), O += P V with P as the TMEM operand.
//   warps 0-3, 4-7   softmax of chain 0 and chain 1 (a thread owns a row; also writes the queries and the results)
//   warps 8-11, 12-15  loaders of the keys and of the values: 128 tokens from the paged cache into shared memory
//                    (128-byte swizzle), e4m3 codes converted to fp16 on the way
//   warp 16          TMEM; one thread issues the products
//   warp 17          one thread works out the CTA's segments
//   warps 18, 19     plan the token tiles ahead of the loaders: block table, row offsets, rows on their way into L2; then scales
// Registers are dealt out accordingly: 112 for a softmax thread, 88 for a loader's, 80 for the others.  Between them the
// roles' loops have to stay in the SM's instruction cache (with twice the unrolling every role ran at half its speed):
// hence short loops where straight runs would do.
// Two chains keep the tensor core busy while a softmax runs.  Their steps alternate; within a chain, P V of a token tile
// and Q K^T of the chain's next one are issued back to back.
//   "dual" item: more than 128 rows, the chains are rows 0-127 and 128-255 and share every token tile;
//   "single" item: up to 128 rows, the chains take alternate token tiles of the same rows and are merged at the end.
// Work: items are (request, kv head, row tile), and each is worth its request's number of token tiles.  With at least four
// items of 256 rows per CTA, none of them large, a CTA takes whole items from its share of the line (row tiles of a request
// are dealt from both ends, since causal ones get longer); otherwise items have 128 rows and the line is cut evenly, as in paged_attention.cu,
// with the parts joined by the last CTA to arrive.
//
// The running maximum that the rows refer to is only raised when it is exceeded by 2^8, so O rarely has to be scaled
// inside TMEM; P is counted from 2^(6 - E) for fp16 (largest product 2^14, all bits kept down to 2^-20 of the row's
// reference and nothing dropped above 2^-30), E as in paged_attention.cu but -120 at least (2^(6 - E) and 2^(E - 6) are normal
// numbers).
// What bounds it: for many rows the issue of the softmax and of the loaders' conversions beside the tensor core, and the
// instruction cache between them; Q K^T with both operands in shared memory takes all of its bandwidth while it runs.  2 x
// 4096 tokens behind 16384, 32 / 8 heads of 128, e4m3: 2.13 ms, 643 TFLOP/s.  For few rows a tile of 128 tokens takes a
// CTA 4000 to 5500 cycles in any case: 16 requests of 8192 tokens with 20 to 128 rows take 140 to 156 us in e4m3, 119 to 150 us
// in bf16 (4.5 to 3.6 TB/s); verification of 4 tokens (8 ragged requests up to 65000) 112 us.
// Every wait is bounded: one that gives up sets UCMR_DEV_WAIT_TIMEOUT and an abort flag, after which no role waits any more
// and all leave by the usual way.
#include "paged_attention.cuh"

namespace ucmr {

int device_sms();

namespace tile {

enum { kBf16 = 0, kF16 = 1, kE4m3 = 2 };

constexpr int kTok = 128;            // tokens per tile
constexpr int kThreads = 640;         // five warpgroups
constexpr int kWarps = kThreads / 32;
constexpr int kLoaders = 128;         // for the keys, and as many for the values
constexpr int kStages = 2;           // of keys and of values each
constexpr int kMetaSlots = 8;
constexpr int kSegments = 4;         // ring of segments between the scheduler and the other roles
constexpr int kSegmentReaders = 10;  // the softmax warps, the tile planner and the products' thread
constexpr int kTileSlots = 4;        // ring of planned token tiles between the planner and the loaders
constexpr float kLazy = 8.f;         // log2 of how far a row's maximum may rise above its reference
constexpr float kShift = 6.f;
constexpr int kHalfBytes = 128 * 128;  // 128 rows of 64 16-bit values

template <int D> struct Sizes {
    static constexpr int kHalves = D / 64;
    static constexpr int kTileBytes = kHalves * kHalfBytes;   // 128 rows in 16 bits
};

struct Meta {
    float tok[2][kTok];              // scales per token, keys and values, for a tile whose scales do not come down to one
    uint32_t valid[4];
    float scale[2];                  // scale of the whole tile; values: 0 if there is nothing but zeros
    int general[2];                  // the scales per token are in use instead
    int bad;                         // tokens before the end are missing
};

// Sixteen bytes if `on`, zeros otherwise; `swap`: the two halves in the other order.
__device__ __forceinline__ uint4 load_if(const unsigned char* p, bool on, bool swap)
{
    uint4 v;
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
        "@q ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%4];\n\t"
        "@q ld.global.nc.L1::no_allocate.v2.u32 {%2, %3}, [%6];\n\t}"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
        : "l"(p + (swap ? 8 : 0)), "r"((uint32_t)on), "l"(p + (swap ? 0 : 8)));
    return v;
}

// What the loaders have to know of a token tile.
struct TileSlot {
    int64_t off[2][kTok];            // byte offsets of the tokens' rows, keys and values; -1 = nothing there
    int block[kTok];                 // their blocks; -1 = nothing there
    int head, bad;                   // kv head; tokens before the end are missing
    uint32_t fold[2][kTok];          // a token's scale over its tile's, twice in fp16
    int edge;                        // first token if some of the item's rows see the tile's tokens and some do not, else kNoEdge
    int seen;                        // tokens that all rows see
    int folds[2];                    // the quotients are in use
    int end;                         // no tile: the last slot
};
constexpr int kNoEdge = 0x7fffffff;
constexpr uint32_t kNothing = 0xffffffffu;   // scale of a token without a block (a NaN that no arithmetic makes)

// A stretch of an item's token tiles.
struct Segment {
    int b, h, q0;
    int row0, n_rows;           // rows [row0, row0 + 128 or 256) of the request's n_rows
    int first, n;               // token tiles that are computed: first .. first + n - 1; n < 0: no more segments
    int dual;
    int len, nq;
    int min_limit, max_limit;   // fewest and most tokens that one of the item's rows sees
    int c0, c1;                 // CTAs that share the item
    int once;                   // no other item reads the same tokens: they are not in L2 yet
};

template <int D>
struct Shared {
    alignas(1024) unsigned char q[2][Sizes<D>::kTileBytes];
    alignas(1024) unsigned char k[kStages][Sizes<D>::kTileBytes];
    alignas(1024) unsigned char v[kStages][Sizes<D>::kTileBytes];
    Meta meta[kMetaSlots];
    TileSlot tile[kTileSlots];
    int entry[2][kTok];              // block-table entries of the tile to be placed and of the one after
    float merge_m[128], merge_l[128];
    alignas(8) uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t s_full[2], p_full[2], o_full[2], q_full;
    uint64_t seg_full[kSegments], seg_empty[kSegments], t_full[kTileSlots], t_empty[kTileSlots], t_placed[kTileSlots];
    Segment seg[kSegments];
    unsigned long long sums[2][kWarps];
    unsigned long long start_units;
    int start_b;
    uint32_t tmem;
    int last;
    volatile int odd;                // a value above a diagonal that is not finite was taken out of a product
    volatile int abort;
};

__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr)
{
    // rows of 128 bytes, 128-byte swizzle; 1024 bytes between groups of eight rows
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr)
{
    // the same bytes read along the rows: leading offset = next 64 columns, stride offset = next eight rows (tokens)
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(kHalfBytes >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

template <int C>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major)
{
    const uint32_t fmt = C == kBf16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
                 : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
                 : "memory");
}
// Two float32 at a time.
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ uint64_t pairf(float lo, float hi) { return pair(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float2 unpair(uint64_t v)
{
    uint32_t lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
    return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}

// Bounded waits: a number of tries, each of which the hardware may stretch from some 20 ns to a microsecond or so (a tenth of
// a second to a few seconds in all) - no clock is read, since these few instructions stand in every loop of every role, and
// the roles share the instruction cache.
constexpr uint32_t kTries = 1u << 22;

// After a time-out, here or in another role, nothing waits any more.
template <int D>
__device__ __forceinline__ void wait(Shared<D>& sm, uint64_t* bar, uint32_t parity, int32_t* status)
{
#pragma unroll 1
    for (uint32_t n = 0; !mbar_try_wait(bar, parity); ++n) {
        if (sm.abort) return;
        if (n > kTries) {
            sm.abort = 1;
            flag_status(status, UCMR_DEV_WAIT_TIMEOUT);
        }
    }
}

// Wait in the rings of segments and planned tiles, which keep turning when the rest has given up: the abort flag does not
// end it, so that no role reads what another has not finished with.
template <int D>
__device__ __forceinline__ void wait_ring(Shared<D>& sm, uint64_t* bar, uint32_t parity, int32_t* status)
{
#pragma unroll 1
    for (uint32_t n = 0; !mbar_try_wait(bar, parity); ++n) {
        if (n > 8 * kTries) {
            sm.abort = 1;
            flag_status(status, UCMR_DEV_WAIT_TIMEOUT);
            return;
        }
    }
}

__device__ __forceinline__ void copy4(void* dst, const void* src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

template <int C>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if constexpr (C == kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(h);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(h);
    }
}
__device__ __forceinline__ float2 unpack2(uint32_t v, bool bf16)
{
    if (bf16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return __half22float2(reinterpret_cast<const __half2&>(v));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
    return r;
}

// Where 16-byte piece `c` (0..7) of 64-column half `half` of a row lies in a swizzled tile.
__device__ __forceinline__ uint32_t swz(int half, int row, int c)
{
    return (uint32_t)half * kHalfBytes + (uint32_t)row * 128u + (uint32_t)((c ^ (row & 7)) << 4);
}

struct Line {
    unsigned long long total, n_cta, u0, u1;
    int rows;      // rows per item: 256 (whole items) or 128 (cut evenly)
};

// An item counts its token tiles, and kItemCost more for reading its queries and writing its rows (about 10 us, where a
// tile of 128 rows takes 2 to 3).
constexpr int kItemCost = 4;
__device__ __forceinline__ int tiles_in(const AttnRequest& r) { return max(1, (r.len + kTok - 1) / kTok); }
__device__ __forceinline__ int units_of(const AttnRequest& r) { return tiles_in(r) + kItemCost; }
__device__ __forceinline__ int tiles_of(const AttnParams& p, const AttnRequest& r, int rows)
{
    return (int)(((int64_t)r.nq * p.G + rows - 1) / rows);
}
__device__ __forceinline__ unsigned long long line_of(const AttnParams& p, int b, int rows)
{
    const AttnRequest r = attn_request(p, b);
    return (unsigned long long)units_of(r) * (unsigned)tiles_of(p, r, rows) * (unsigned)p.Hkv;
}

// Next segment of the CTA's stretch of the line; n < 0 at its end.
struct SegmentWalk {
    int b;
    unsigned long long b_first, u;

    __device__ __forceinline__ void next(const AttnParams& p, const Line& line, Segment& s)
    {
        for (;;) {
            s.n = -1;
            if (u >= line.u1) return;
            AttnRequest r;
            int tiles, units;
            for (;;) {
                if (b >= p.B) return;  // (lengths that changed under the kernel)
                r = attn_request(p, b);
                units = units_of(r);
                tiles = tiles_of(p, r, line.rows);
                const unsigned long long n = (unsigned long long)units * (unsigned)tiles * (unsigned)p.Hkv;
                if (u < b_first + n) break;
                b_first += n;
                ++b;
            }
            const unsigned long long in_b = u - b_first;
            const int item = (int)(in_b / units);
            const int from = (int)(in_b - (unsigned long long)item * units);
            const unsigned long long item_first = u - from;
            const int in_item = tiles_in(r);
            int to = in_item;
            u = item_first + units;
            s.c0 = s.c1 = blockIdx.x;
            if (line.rows == 256) {
                if (from != 0) continue;  // an item belongs to the CTA in whose stretch it begins
            } else {
                if (from >= in_item) continue;
                to = (int)min((unsigned long long)in_item, line.u1 - item_first);
                s.c0 = (int)(((item_first + 1) * line.n_cta - 1) / line.total);
                s.c1 = (int)(((item_first + in_item) * line.n_cta - 1) / line.total);
            }
            s.b = b;
            s.q0 = r.q0; s.len = r.len; s.nq = r.nq;
            s.h = item / tiles;
            const int at = item - s.h * tiles;
            const int rt = (at & 1) ? tiles - 1 - (at >> 1) : at >> 1;
            s.n_rows = r.nq * p.G;
            s.row0 = rt * line.rows;
            const int last_row = min(s.n_rows, s.row0 + line.rows) - 1;
            s.once = tiles == 1;
            s.dual = last_row - s.row0 >= 128;
            s.min_limit = attn_limit(p, r, s.row0 / p.G);
            s.max_limit = attn_limit(p, r, last_row / p.G);
            s.first = from;
            s.n = max(0, min(to, (s.max_limit + kTok - 1) / kTok) - from);
            return;
        }
    }
};

template <int D, int C, typename QT>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const __grid_constant__ AttnParams p)
{
    extern __shared__ unsigned char s_raw[];
    Shared<D>& sm = *reinterpret_cast<Shared<D>*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    constexpr bool kQBf16 = __is_same(QT, __nv_bfloat16);
    constexpr int kP = C == kBf16 ? kBf16 : kF16;      // type of the products' operands
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float inf = __uint_as_float(0x7f800000u);

    // ---- set-up: barriers, TMEM, the CTA's stretch of the line -------------------------------------------------------
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sm.k_full[i], kLoaders / 32); mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_full[i], kLoaders / 32); mbar_init(&sm.v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(&sm.s_full[i], 1); mbar_init(&sm.p_full[i], 4); mbar_init(&sm.o_full[i], 1); }
        for (int i = 0; i < kSegments; ++i) { mbar_init(&sm.seg_full[i], 1); mbar_init(&sm.seg_empty[i], kSegmentReaders); }
        for (int i = 0; i < kTileSlots; ++i) { mbar_init(&sm.t_full[i], 1); mbar_init(&sm.t_placed[i], 1); mbar_init(&sm.t_empty[i], 2 * kLoaders / 32); }
        mbar_init(&sm.q_full, 8);
        sm.abort = 0;
        sm.odd = 0;
        fence_mbar_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int per = (p.B + kThreads - 1) / kThreads;
    unsigned long long mine[2] = {0, 0}, before[2];
    unsigned long long whole_items = 0;
    int largest = 0;
    for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) {
        mine[0] += line_of(p, b, 128);
        mine[1] += line_of(p, b, 256);
        const AttnRequest r = attn_request(p, b);
        whole_items += (unsigned long long)tiles_of(p, r, 256) * (unsigned)p.Hkv;
        if (r.nq > 0) largest = max(largest, units_of(r));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        before[k] = mine[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long v = __shfl_up_sync(0xffffffffu, before[k], o);
            if (lane >= o) before[k] += v;
        }
        if (lane == 31) sm.sums[k][warp] = before[k];
    }
    fence_before();
    __syncthreads();
    fence_after();
    unsigned long long total[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        unsigned long long offset = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) offset += sm.sums[k][w];
            total[k] += sm.sums[k][w];
        }
        before[k] += offset - mine[k];
    }
    __syncthreads();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) whole_items += __shfl_xor_sync(0xffffffffu, whole_items, o);
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (lane == 0) { sm.sums[0][warp] = whole_items; sm.sums[1][warp] = largest; }
    __syncthreads();
    whole_items = 0;
    for (int w = 0; w < kWarps; ++w) { whole_items += sm.sums[0][w]; largest = max(largest, (int)sm.sums[1][w]); }
    Line line;
    // whole items of 256 rows: at least four per CTA, and none that takes more than a third of a CTA's share
    const int kind = whole_items >= 4ull * gridDim.x && 3ull * largest * gridDim.x <= total[1] ? 1 : 0;
    line.rows = kind ? 256 : 128;
    line.total = total[kind];
    line.n_cta = min((unsigned long long)gridDim.x, line.total);
    const bool idle = blockIdx.x >= line.n_cta;
    line.u0 = idle ? 0 : blockIdx.x * line.total / line.n_cta;
    line.u1 = idle ? 0 : (blockIdx.x + 1) * line.total / line.n_cta;
    if (!idle && before[kind] <= line.u0 && line.u0 < before[kind] + mine[kind]) {
        unsigned long long at = before[kind];
        for (int b = tid * per; b < p.B; ++b) {
            const unsigned long long n = line_of(p, b, line.rows);
            if (line.u0 < at + n) { sm.start_b = b; sm.start_units = at; break; }
            at += n;
        }
    }
    __syncthreads();
    const uint32_t tmem = sm.tmem;
    // columns: S (and P) of chain T at 128 T, O at 256 + 128 T
    auto tS = [&](int T) { return tmem + T * 128; };
    auto tO = [&](int T) { return tmem + 256 + T * 128; };
    uint32_t n_seg = 0;
    auto take_segment = [&]() -> const Segment& {
        wait_ring(sm, &sm.seg_full[n_seg % kSegments], (n_seg / kSegments) & 1, p.status);
        return sm.seg[n_seg % kSegments];
    };
    auto drop_segment = [&]() { mbar_arrive(&sm.seg_empty[n_seg % kSegments]); ++n_seg; };  // (one thread per reader)

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        // ================================= softmax ================================================================
        const int T = warp >> 2;                   // chain
        const int local = (warp & 3) * 32 + lane;  // row of the tile = TMEM lane
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        uint32_t n_s = 0, n_o = 0;                 // phases seen
        uint32_t tile0 = 0;                        // token tiles of the CTA before this segment
        for (;;) {
            const Segment s = take_segment();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.seg_empty[n_seg % kSegments]);
            ++n_seg;
            if (s.n < 0) break;
            const AttnRequest request = {s.len, s.q0, s.nq};
            const int row = s.row0 + (s.dual ? T * 128 : 0) + local;
            const bool live = row < s.n_rows;
            const int steps = s.dual ? s.n : (s.n + 1 - T) / 2;   // of this chain
            float qmul = p.scale_log2;
            // queries: this thread's row, 16-bit, swizzled (single: chain 0 writes the tile that both chains read)
            if (s.n > 0 && (s.dual || T == 0)) {
                const QT* qr = static_cast<const QT*>(p.q);
                if (live) qr += (int64_t)(s.q0 + row / p.G) * p.qs_t + (int64_t)(s.h * p.G + row % p.G) * p.qs_h;
                uint4 v[D / 8];                      // (all loads at once)
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    v[c] = make_uint4(0, 0, 0, 0);
                    if (live) v[c] = *reinterpret_cast<const uint4*>(qr + c * 8);
                }
                float down = 1.f;
                if constexpr (C == kE4m3) {
                    uint32_t m2 = 0;                 // largest magnitudes of the even and odd elements, as 16-bit patterns
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        m2 = __vmaxu2(m2, v[c].x & 0x7fff7fffu); m2 = __vmaxu2(m2, v[c].y & 0x7fff7fffu);
                        m2 = __vmaxu2(m2, v[c].z & 0x7fff7fffu); m2 = __vmaxu2(m2, v[c].w & 0x7fff7fffu);
                    }
                    const float2 m = unpack2(m2, kQBf16);
                    uint32_t big = __float_as_uint(fmaxf(m.x, m.y));
                    if (!(m.x <= 3.402823466e38f && m.y <= 3.402823466e38f)) big = 0;   // (the row is not finite: nor is its result)
                    const int e = big == 0 ? 0 : max(-125, min(125, (int)(big >> 23) - 127));
                    down = __uint_as_float((uint32_t)(127 - e) << 23);
                    if (!s.dual) sm.merge_m[local] = __uint_as_float((uint32_t)(127 + e) << 23);
                    qmul *= __uint_as_float((uint32_t)(127 + e) << 23);
                }
                unsigned char* dst = sm.q[s.dual ? T : 0];
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    if constexpr (C == kE4m3) {
                        uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 f = unpack2(w[i], kQBf16);
                            w[i] = pack2<kF16>(f.x * down, f.y * down);
                        }
                        v[c] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    *reinterpret_cast<uint4*>(dst + swz(c >> 3, local, c & 7)) = v[c];
                }
                fence_proxy_async();
            }
            if (s.n > 0) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.q_full);
                if (C == kE4m3 && !s.dual) {
                    bar_sync(1, 256);
                    if (T == 1) qmul *= sm.merge_m[local];
                    bar_sync(1, 256);  // (merge_m is used again)
                }
            }
            const int limit = live ? attn_limit(p, request, row / p.G) : s.max_limit;
            const int warp_limit = __reduce_min_sync(0xffffffffu, limit);
            float ref = -inf, sum = 0.f;
            int vexp = -200;
            float vf_of = 0.f, vf_log = 0.f, vf_inv = 1.f;       // a factor on the weights, its logarithm and reciprocal
            for (int st = 0; st < steps; ++st) {
                const int i = s.dual ? st : 2 * st + T;          // token tile of the segment
                const int tok0 = (s.first + i) * kTok;
                wait(sm, &sm.s_full[T], n_s & 1, p.status);
                ++n_s;
                fence_after();
                const Meta& mt = sm.meta[(tile0 + i) % kMetaSlots];
                const uint32_t tS_at = tS(T) + lane_at;
                float kf = qmul, vf = C == kBf16 ? 1.f : 64.f;
                float vdown = 1.f;
                bool kgen = false, vgen = false;
                if constexpr (C == kE4m3) {
                    const float vscale = mt.scale[1];
                    kgen = mt.general[0] != 0;
                    vgen = mt.general[1] != 0;
                    if (!kgen) kf *= mt.scale[0];
                    if (__float_as_uint(vscale) == 0) {              // no values but zeros, in the product too: no say in E
                        vf = 1.f;
                    } else {
                        const int e = max(-120, min(128, (int)((__float_as_uint(vscale) & 0x7fffffffu) >> 23) - 126));
                        if (e > vexp) {
                            vdown = vexp == -200 ? 0.f : exp2_fast((float)(vexp - e));
                            vexp = e;
                        }
                        vf = exp2_fast(kShift - (float)vexp);
                        if (!vgen) vf *= vscale;
                    }
                }
                // One scale, and no token missing but at the end: columns from `bound` on are hidden.  The factor on the weights
                // goes into their exponential and is taken out of their sum again: not where it is so small that weights
                // which the sum needs would vanish (at 2^-60 those below 2^-66 of the reference do).  A warp goes one way as a
                // whole, since both read the tensor memory together: the factor of a row of tiny queries may be 0 alone.
                const bool plain = __all_sync(0xffffffffu, !kgen && !vgen && kf > 0.f && vf >= 0x1p-60f && !mt.bad);
                const int bound = limit - tok0;
                float alpha = 1.f;
                auto raise = [&](float top) {
                    if (top > ref + kLazy || (ref == -inf && top > -inf)) {
                        alpha = exp2_fast(ref - top);  // (0 from -inf)
                        ref = top;
                        sum *= alpha;
                    }
                    if (st > 0 && __any_sync(0xffffffffu, alpha != 1.f || vdown != 1.f)) {
                        const float f = alpha * vdown;
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t r[16];
                            ld16(tO(T) + lane_at + c * 16, r);
                            wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f);
                            st16(tO(T) + lane_at + c * 16, r);
                        }
                    }
                };
                if (plain) {
                    const bool cut = tok0 + kTok > warp_limit;
                    uint32_t r[32];
                    auto fetch = [&](int c) {        // columns 32c ..; hidden ones -> no weight
                        ld32(tS_at + c * 32, r);
                        wait_ld();
                        if (cut) {
                            const int from = bound - c * 32;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j >= from) r[j] = 0xff800000u;
                        }
                    };
                    float t4[4] = {-inf, -inf, -inf, -inf};
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        fetch(c);
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            t4[(j >> 1) & 3] = max3(t4[(j >> 1) & 3], __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
                    }
                    raise(fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * kf);
                    // exp2(score - reference) * vf in one exponential; the sum is taken back to weights at the end.  P of
                    // columns 32c.. goes to 64 + 16c..: from the last ones down no column is overwritten before it is read.
                    if (C != kBf16 && vf != vf_of) {
                        vf_of = vf;
                        vf_log = log2f(vf);
                        vf_inv = 1.f / vf;
                    }
                    const float base = vf_log - (ref == -inf ? 0.f : ref);
                    const uint64_t kf2 = pairf(kf, kf), base2 = pairf(base, base);
                    uint64_t acc[2] = {0, 0};
#pragma unroll 1
                    for (int c = 3; c >= 0; --c) {
                        uint32_t w[16];
                        fetch(c);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 x = unpair(fma2(pair(r[j], r[j + 1]), kf2, base2));
                            const float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
                            acc[(j >> 1) & 1] = add2(acc[(j >> 1) & 1], pairf(e0, e1));
                            w[j / 2] = pack2<kP>(e0, e1);
                        }
                        st16(tS_at + 64 + c * 16, w);
                    }
                    const float2 a = unpair(add2(acc[0], acc[1]));
                    sum += (a.x + a.y) * vf_inv;
                } else {
                    float top = -inf;
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        uint32_t r[16];
                        ld16(tS_at + c * 16, r);
                        wait_ld();
                        const uint32_t seen16 = mt.valid[c >> 1] >> ((c & 1) * 16);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            float x = __uint_as_float(r[j]) * kf;
                            if (kgen) x *= mt.tok[0][c * 16 + j];
                            top = tok0 + c * 16 + j < limit && ((seen16 >> j) & 1u) ? fmaxf(top, x) : top;
                        }
                    }
                    raise(top);
                    const float base = ref == -inf ? 0.f : ref;
                    // P of columns 16c.. goes to 64 + 8c..; in this order no column is overwritten before it is read:
                    // 7 -> 120.., 6 -> 112.., 5 -> 104.., 4 -> 96.., then 3 -> 88.. down to 0 -> 64..
#pragma unroll 1
                    for (int c = 7; c >= 0; --c) {
                        uint32_t r[16], w[8];
                        ld16(tS_at + c * 16, r);
                        wait_ld();
                        const uint32_t seen16 = mt.valid[c >> 1] >> ((c & 1) * 16);
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float x[2];
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                x[q] = __uint_as_float(r[j + q]) * kf;
                                if (kgen) x[q] *= mt.tok[0][c * 16 + j + q];
                                const bool seen = tok0 + c * 16 + j + q < limit && ((seen16 >> (j + q)) & 1u);
                                x[q] = seen ? exp2_fast(x[q] - base) : 0.f;
                                sum += x[q];
                                if (!vgen) x[q] *= vf;
                                else x[q] = seen ? x[q] * (vf * mt.tok[1][c * 16 + j + q]) : 0.f;   // (vf alone may reach 2^126)
                            }
                            w[j / 2] = pack2<kP>(x[0], x[1]);
                        }
                        st8(tS_at + 64 + c * 8, w);
                    }
                }
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_full[T]);
            }
            // ---- results ---------------------------------------------------------------------------------------------
            if (steps > 0) {
                wait(sm, &sm.o_full[T], n_o & 1, p.status);
                ++n_o;
                fence_after();
            }
            float unit = C == kBf16 ? 1.f : exp2_fast((C == kE4m3 && vexp != -200 ? (float)vexp : 0.f) - kShift);
            bool holds = steps > 0;                 // O of this chain has been written
            float mine_f = 1.f, other_f = 0.f;      // single: factors of the two chains
            float* other = reinterpret_cast<float*>(sm.q[0]);   // chain 1's rows, in the place of the queries
            if (!s.dual) {
                if (T == 1) {
                    sm.merge_m[local] = ref;
                    sm.merge_l[local] = sum;
                }
                bar_sync(1, 256);  // also: both chains' products are done, the queries are free
                if (T == 1 && holds) {
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t r[16];
                        ld16(tO(1) + lane_at + c * 16, r);
                        wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const int piece = c * 4 + j / 4;
                            *reinterpret_cast<float4*>(other + local * D + ((piece ^ (local & (D / 4 - 1))) * 4)) =
                                make_float4(__uint_as_float(r[j]) * unit, __uint_as_float(r[j + 1]) * unit,
                                            __uint_as_float(r[j + 2]) * unit, __uint_as_float(r[j + 3]) * unit);
                        }
                    }
                }
                bar_sync(1, 256);
                if (T == 0) {
                    const float m1 = sm.merge_m[local], l1 = sm.merge_l[local];
                    const float m = fmaxf(ref, m1);
                    mine_f = ref == -inf ? 0.f : exp2_fast(ref - m);
                    other_f = m1 == -inf ? 0.f : exp2_fast(m1 - m);
                    sum = (ref == -inf ? sum : sum * mine_f) + (m1 == -inf ? l1 : l1 * other_f);
                    ref = m;
                }
            }
            const bool writer = s.dual || T == 0;
            const int c0 = s.c0, c1 = s.c1;
            const bool whole = c0 == c1;
            constexpr int kRowFloats = D + 2;
            float* part = p.partial + ((int64_t)blockIdx.x * 2 + ((int)blockIdx.x == c0 ? 1 : 0)) * 128 * kRowFloats;
            const float inv = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
            const int64_t tok = s.q0 + row / p.G;
            const int head = s.h * p.G + row % p.G;
            const bool odd = sm.odd != 0;
            if (writer) {
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    __syncwarp();   // (rows that are not there have gone ahead)
                    float o[16];
                    if (holds) {
                        uint32_t r[16];
                        ld16(tO(T) + lane_at + c * 16, r);
                        wait_ld();
                        // (a chain without a finite reference holds zeros, or NaN that its sum has too)
                        const float f = s.dual ? unit : unit * mine_f;
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = (s.dual ? ref : mine_f) == (s.dual ? -inf : 0.f) ? 0.f : __uint_as_float(r[j]) * f;
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = 0.f;
                    }
                    if (!s.dual && s.n > 1) {
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const int piece = c * 4 + j / 4;
                            const float4 x = *reinterpret_cast<const float4*>(other + local * D + ((piece ^ (local & (D / 4 - 1))) * 4));
                            if (other_f != 0.f) {
                                o[j] += other_f * x.x; o[j + 1] += other_f * x.y;
                                o[j + 2] += other_f * x.z; o[j + 3] += other_f * x.w;
                            }
                        }
                    }
                    if (odd && live) {
                        // values above the diagonal that are not finite were taken out of the product: back to the rows that see them
                        const int from = max(s.min_limit, s.first * kTok), to = min(limit, (s.first + s.n) * kTok);
#pragma unroll 1
                        for (int tk = from; tk < to; ++tk) {
                            const int blk = p.table[(int64_t)s.b * p.bt_b + (int64_t)s.h * p.bt_h + p.by_block.div(tk)];
                            if (blk < 0 || blk >= p.NB) continue;
                            const unsigned char* vr = static_cast<const unsigned char*>(p.cache[1]) + blk * p.cs_b[1] +
                                                      (int64_t)(tk - p.by_block.div(tk) * p.BS) * p.cs_t[1] + s.h * p.cs_h[1];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const int d = c * 16 + j;
                                if constexpr (C == kE4m3) {
                                    if ((vr[d] & 0x7fu) == 0x7fu) o[j] += __uint_as_float(0x7fffffffu);
                                } else {
                                    const uint16_t h16 = reinterpret_cast<const uint16_t*>(vr)[d];
                                    const float x = unpack2(h16, C == kBf16).x;
                                    if (!(fabsf(x) <= 3.402823466e38f)) o[j] += x;
                                }
                            }
                        }
                    }
                    if (!live) continue;
                    if (whole) {
                        QT* dst = static_cast<QT*>(p.out) + tok * p.os_t + (int64_t)head * p.os_h + c * 16;
#pragma unroll
                        for (int j = 0; j < 16; j += 8) {
                            uint4 v;
                            constexpr int kO = kQBf16 ? kBf16 : kF16;
                            v.x = pack2<kO>(o[j] * inv, o[j + 1] * inv);     v.y = pack2<kO>(o[j + 2] * inv, o[j + 3] * inv);
                            v.z = pack2<kO>(o[j + 4] * inv, o[j + 5] * inv); v.w = pack2<kO>(o[j + 6] * inv, o[j + 7] * inv);
                            *reinterpret_cast<uint4*>(dst + j) = v;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j += 4)
                            *reinterpret_cast<float4*>(part + local * D + c * 16 + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
                if (live) {
                    if (whole) {
                        if (p.lse != nullptr) p.lse[tok * p.Hq + head] = sum == 0.f ? -inf : (ref + log2f(sum)) * 0.69314718055994531f;
                    } else {
                        part[128 * D + local] = ref;
                        part[128 * (D + 1) + local] = sum;
                    }
                }
            }
            fence_before();   // O and S are read; the next products may overwrite them once the queries are announced
            if (!whole) {
                __threadfence();
                bar_sync(1, 256);
                if (tid == 0) {
                    const int old = atom_add_release_gpu(p.counters + c0, 1);
                    sm.last = old == c1 - c0;
                    if (sm.last) p.counters[c0] = 0;
                }
                bar_sync(1, 256);
                if (sm.last) {
                    __threadfence();
                    attn_join<D, 128, 8, false, QT>(p, c0, c1, min(128, s.n_rows - s.row0), warp, lane, nullptr, [&](int r, int64_t& to, int& of) {
                        to = s.q0 + (s.row0 + r) / p.G;
                        of = s.h * p.G + (s.row0 + r) % p.G;
                        return true;
                    });
                }
            }
            bar_sync(1, 256);  // the queries and the merged rows have been used
            tile0 += s.n;
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // ================================= loaders ================================================================
        constexpr int kEs = C == kE4m3 ? 1 : 2;
        constexpr int kPer = D * kEs / 16;           // 16-byte pieces per row
        constexpr int kRows = kLoaders / kPer;       // rows per pass
        constexpr int kPasses = kTok / kRows;
        const int kind = warp < 12 ? 0 : 1;          // keys, values
        const int lt = tid - 256 - kind * kLoaders;
        const int piece = lt % kPer, prow = lt / kPer;
        uint64_t* full = kind ? sm.v_full : sm.k_full;
        uint64_t* empty = kind ? sm.v_empty : sm.k_empty;
        unsigned char* ring = kind ? sm.v[0] : sm.k[0];
        const unsigned char* cache = static_cast<const unsigned char*>(p.cache[kind]);
        uint32_t done = 0;                           // token tiles of the CTA so far: stage = done % 2
        // (The fence between these writes and the products' reads is with the reader, after its wait: here it would also wait
        // for the loads that are under way.)
        auto arrive = [&](uint64_t* b) {
            __syncwarp();
            if (lane == 0) mbar_arrive(b);
        };

        // Values of a tile that only some rows see, where they are not finite: out of the product (the epilogue gives them
        // to the rows that see them).  A thread looks at what it has written itself.
        auto sift = [&](int st, int edge, int seen) {
            bool odd = false;
            constexpr uint32_t kExp = C == kBf16 ? 0x7f80u : 0x7c00u;
            constexpr int kHere = D / 8;               // 16-byte pieces per row in shared memory
            constexpr int kOwn = C == kE4m3 ? 2 : 1;   // of which this thread wrote so many, side by side
#pragma unroll 1
            for (int i = 0; i < kPasses * kOwn; ++i) {
                const int row = i / kOwn * kRows + prow, c = piece * kOwn + i % kOwn;
                static_assert(kHere == kPer * kOwn, "pieces");
                if (edge + row < seen) continue;
                uint32_t* at = reinterpret_cast<uint32_t*>(ring + st * Sizes<D>::kTileBytes + swz(c >> 3, row, c & 7));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = at[j];
                    uint32_t n = w;
                    if ((w & kExp) == kExp) n &= 0xffff0000u;
                    if (((w >> 16) & kExp) == kExp) n &= 0xffffu;
                    if (n != w) { at[j] = n; odd = true; }
                }
            }
            if (odd) sm.odd = 1;
        };

        auto slot_at = [&](uint32_t tile) -> const TileSlot& {   // waits until the tile has been planned
            wait_ring(sm, &sm.t_full[tile % kTileSlots], (tile / kTileSlots) & 1, p.status);
            return sm.tile[tile % kTileSlots];
        };
        auto planned = [&](uint32_t tile) { return mbar_test_wait(&sm.t_full[tile % kTileSlots], (tile / kTileSlots) & 1); };
        auto drop_slot = [&](uint32_t tile) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.t_empty[tile % kTileSlots]);
        };
        if constexpr (C == kE4m3) {
            // A tile of codes waits in registers; each piece's place is taken by the next tile's as soon as it is stored.
            // Sixteen codes -> two 16-byte pieces; half of the lanes take them in the other order, so that the lanes of a
            // row, which hold both column halves, do not meet in a bank.
            const int flip = (piece >> 2) & 1, c0 = (piece & 3) * 2;
            uint4 raw[kPasses];
            // has: a tile is in registers; more: the next one's rows are known.  If they are not yet, the tile in hand goes out
            // without waiting for them: the planner may itself be waiting for what follows from it.
            bool has = false, ended = false;
            for (;;) {
                bool more = false;
                if (!ended) {
                    more = true;
                    if (has) more = __all_sync(0xffffffffu, planned(done + 1));
                    else slot_at(done);
                }
                const TileSlot& next = sm.tile[(done + has) % kTileSlots];
                if (more && next.end) { more = false; ended = true; }
                if (!has && !more) break;
                const int st = done % kStages;
                const TileSlot& slot = sm.tile[done % kTileSlots];
                if (has) wait(sm, &empty[st], ((done / kStages) & 1) ^ 1, p.status);
                if (has) {
                    // rows i * kRows + prow: the swizzle of a row depends on row % 8, which all of a thread's rows share
                    unsigned char* dst = ring + st * Sizes<D>::kTileBytes;
                    unsigned char* d0 = dst + swz(piece >> 2, prow, c0 + flip);
                    unsigned char* d1 = dst + swz(piece >> 2, prow, c0 + 1 - flip);
                    static_assert(kRows % 8 == 0, "swizzle");
                    const bool folds = slot.folds[kind] != 0;
#pragma unroll
                    for (int i = 0; i < kPasses; ++i) {
                        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                        uint32_t f[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) f[j] = e4m3x2_to_f16x2(j & 1 ? w[j >> 1] >> 16 : w[j >> 1]);
                        if (folds) {
                            const uint32_t mw = slot.fold[kind][i * kRows + prow];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const __half2 v = __hmul2(reinterpret_cast<const __half2&>(f[j]), reinterpret_cast<const __half2&>(mw));
                                f[j] = reinterpret_cast<const uint32_t&>(v);
                            }
                        }
                        const uint4 a = make_uint4(f[0], f[1], f[2], f[3]), b = make_uint4(f[4], f[5], f[6], f[7]);
                        *reinterpret_cast<uint4*>(d0 + i * kRows * 128) = a;
                        *reinterpret_cast<uint4*>(d1 + i * kRows * 128) = b;
                    }
                    if (kind == 1 && slot.edge != kNoEdge) sift(st, slot.edge, slot.seen);
                    arrive(&full[st]);
                }
                if (more) {
#pragma unroll
                    for (int i = 0; i < kPasses; ++i) {
                        const int64_t off = next.off[kind][i * kRows + prow];
                        raw[i] = load_if(cache + off + piece * 16, off >= 0, flip != 0);
                    }
                }
                if (has) drop_slot(done++);
                has = more;
            }
        } else {
            // 16-bit rows go straight into the swizzled tiles.  A tile is announced once the next one has been asked for, or
            // at once if there is no room for that yet.
            bool owed = false;
            for (;;) {
                const int st = done % kStages;
                const uint32_t parity = ((done / kStages) & 1) ^ 1;
                if (owed && !__all_sync(0xffffffffu, planned(done) && mbar_test_wait(&empty[st], parity))) {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    arrive(&full[st ^ 1]);
                    owed = false;
                }
                const TileSlot& slot = slot_at(done);
                if (slot.end) break;
                wait(sm, &empty[st], parity, p.status);
                const uint32_t d0 = smem_u32(ring + st * Sizes<D>::kTileBytes);
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const int row = i * kRows + prow;
                    const int64_t off = slot.off[kind][row];
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d0 + swz(piece >> 3, row, piece & 7)),
                                 "l"(off >= 0 ? cache + off + piece * 16 : cache), "r"(off >= 0 ? 16 : 0)
                                 : "memory");
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (owed) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    arrive(&full[st ^ 1]);
                }
                owed = true;
                if (kind == 1 && slot.edge != kNoEdge) {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    sift(st, slot.edge, slot.seen);
                }
                drop_slot(done);
                ++done;
            }
            if (owed) {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                arrive(&full[(done - 1) % kStages]);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // ================================= products ===============================================================
        if (warp == 16 && lane == 0) {
        uint32_t tiles = 0;                 // token tiles before this segment
        uint32_t n_p = 0, n_q = 0;          // phases seen (a bit per chain)
        for (;;) {
            const Segment& slot = take_segment();
            const int s_n = slot.n;
            const bool dual = slot.dual != 0;
            drop_segment();
            if (s_n < 0) break;
            if (s_n == 0) continue;
            const int steps = dual ? 2 * s_n : s_n;
            auto scores = [&](int st) {
                const int i = dual ? st >> 1 : st, T = st & 1;
                const uint32_t tile = tiles + i, stage = tile % kStages;
                if (!dual || T == 0) {
                    wait(sm, &sm.k_full[stage], (tile / kStages) & 1, p.status);
                    fence_proxy_async();
                }
                const uint64_t qa = desc_k_major(smem_u32(sm.q[dual ? T : 0])), ka = desc_k_major(smem_u32(sm.k[stage]));
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    constexpr int kStep = 32 >> 4, kHalf = kHalfBytes >> 4;   // (descriptors count 16-byte units)
                    const uint32_t off = (ks >> 2) * kHalf + (ks & 3) * kStep;
                    mma_ss(tS(T), qa + off, ka + off, idesc<kP>(kTok, false), ks > 0);
                }
                commit(&sm.s_full[T]);
                if (!dual || T == 1) commit(&sm.k_empty[stage]);
            };
            wait(sm, &sm.q_full, n_q & 1, p.status);
            ++n_q;
            fence_after();
            for (int st = -2; st < steps; ++st) {
                const int T = st & 1;
                if (st >= 0) {
                    const int i = dual ? st >> 1 : st;
                    const uint32_t tile = tiles + i, stage = tile % kStages;
                    if (!dual || T == 0) {
                        wait(sm, &sm.v_full[stage], (tile / kStages) & 1, p.status);
                        fence_proxy_async();
                    }
                    wait(sm, &sm.p_full[T], (n_p >> T) & 1, p.status);
                    n_p ^= 1u << T;
                    fence_after();
                    const uint64_t va = desc_mn_major(smem_u32(sm.v[stage]));
                    const bool first = dual ? i == 0 : st < 2;
#pragma unroll
                    for (int ks = 0; ks < kTok / 16; ++ks)
                        mma_ts(tO(T), tS(T) + 64 + ks * 8, va + ks * (2048 >> 4), idesc<kP>(D, true), !first || ks > 0);
                    if (!dual || T == 1) commit(&sm.v_empty[stage]);
                }
                if (st + 2 < steps) scores(st + 2);
                else if (st >= 0) commit(&sm.o_full[T]);
            }
            tiles += s_n;
        }
        } else if (warp == 18) {
            // ============================= places: one token tile at a time, four tokens per lane ==========================
            uint32_t tile = 0;
            for (bool more = true; more;) {
                const Segment& s = take_segment();
                const int n = s.n, first = s.first, low = s.min_limit, high = s.max_limit, h = s.h, once = s.once;
                const int32_t* table = p.table + (int64_t)s.b * p.bt_b + (int64_t)s.h * p.bt_h;
                __syncwarp();
                if (lane == 0) drop_segment();
                else ++n_seg;
                more = n >= 0;
                // The next tile's entries are copied while this one is placed; a lane reads what it has copied itself.
                auto look_up = [&](int i, uint32_t t) {
                    if (i < n) {
#pragma unroll 1
                        for (int at = lane; at < kTok; at += 32) {
                            const int tok = (first + i) * kTok + at;
                            if (tok < high) copy4(&sm.entry[t & 1][at], table + p.by_block.div(tok));
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
                look_up(0, tile);
#pragma unroll 1
                for (int i = 0; i < max(n, more ? 0 : 1); ++i, ++tile) {
                    TileSlot& slot = sm.tile[tile % kTileSlots];
                    look_up(i + 1, tile + 1);
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    wait_ring(sm, &sm.t_empty[tile % kTileSlots], ((tile / kTileSlots) & 1) ^ 1, p.status);
                    if (more) {
                        const int tok0 = (first + i) * kTok;
                        bool missing = false;
#pragma unroll 1
                        for (int at = lane; at < kTok; at += 32) {
                            const int tok = tok0 + at;
                            int blk = tok < high ? sm.entry[tile & 1][at] : -1;
                            if (blk < 0 || blk >= p.NB) {
                                missing |= tok < high;
                                blk = -1;
                            }
                            const int row = tok - p.by_block.div(tok) * p.BS;
                            const int64_t ko = blk * p.cs_b[0] + row * p.cs_t[0] + h * p.cs_h[0];
                            const int64_t vo = blk * p.cs_b[1] + row * p.cs_t[1] + h * p.cs_h[1];
                            slot.block[at] = blk;
                            slot.off[0][at] = blk >= 0 ? ko : -1;
                            slot.off[1][at] = blk >= 0 ? vo : -1;
                            // The row on its way into L2, a few tiles before the loaders ask for it (verification of 4
                            // tokens: 424 -> 323 us); rows that other items read too are there already.
                            if (blk >= 0 && once) {
                                constexpr int kRowBytes = D * (C == kE4m3 ? 1 : 2);
#pragma unroll
                                for (int l = 0; l < kRowBytes; l += 128) {
                                    asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(p.cache[0]) + ko + l));
                                    asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(p.cache[1]) + vo + l));
                                }
                            }
                        }
                        if (missing) flag_status(p.status, UCMR_DEV_BAD_BLOCK_ID);
                        missing = __any_sync(0xffffffffu, missing);
                        if (lane == 0) {
                            slot.head = h;
                            slot.bad = missing;
                            slot.edge = tok0 + kTok > low && low < high ? tok0 : kNoEdge;
                            slot.seen = low;
                            slot.end = 0;
                        }
                    } else if (lane == 0) {
                        slot.end = 1;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.t_placed[tile % kTileSlots]);
                }
            }
        } else if (warp == 19) {
            // ============================= scales: once the tile has been placed ===================================
            // A tile does not wait for the next one to be placed: segments without tiles (rows that see nothing) may follow, more than
            // the ring holds, and then the planner waits for the softmax, which waits for this tile.  Scales come straight into
            // registers (verification 112 us; by copies through shared memory, a tile ahead, 131), in loops over the lane's four
            // tokens that are unrolled, unlike the others.
            // One scale for the tile, keys and values each.  All alike: that one.  Powers of two within 2^15 of one another: the
            // largest, and the codes are multiplied by the quotient on the way to fp16 - exactly, since a code is a multiple
            // of 2^-9 and fp16 holds multiples of 2^-24.  Otherwise the softmax takes the scales token by token.
#pragma unroll 1
            for (uint32_t tile = 0, end = 0; !end; ++tile) {
                wait_ring(sm, &sm.t_placed[tile % kTileSlots], (tile / kTileSlots) & 1, p.status);
                TileSlot& slot = sm.tile[tile % kTileSlots];
                Meta& mt = sm.meta[tile % kMetaSlots];
                end = slot.end;
                if (!end) {
                    if constexpr (C == kE4m3) {
                        float of[2][kTok / 32];      // the lane's four tokens'
#pragma unroll
                        for (int i = 0; i < kTok / 32; ++i) {
                            const int blk = slot.block[lane + 32 * i];
                            of[0][i] = of[1][i] = __uint_as_float(kNothing);
                            if (blk < 0) continue;
                            const int64_t from = (int64_t)blk * p.Hkv + slot.head;
                            of[0][i] = __ldg(p.scale[0] + from);
                            of[1][i] = __ldg(p.scale[1] + from);
                        }
#pragma unroll 1
                        for (int kind = 0; kind < 2; ++kind) {
                            uint32_t lo = 0xffffffffu, hi = 0, odd = 0, zero = 0;
#pragma unroll
                            for (int i = 0; i < kTok / 32; ++i) {
                                const uint32_t b = __float_as_uint(kind ? of[1][i] : of[0][i]);
                                if (b == kNothing) continue;
                                if (b == 0) { zero = 1; continue; }
                                lo = min(lo, b);
                                hi = max(hi, b);
                                odd |= (b & 0x807fffffu) | (b >= 0x7f800000u ? 1u : 0u);   // no power of two, negative, subnormal
                            }
                            lo = __reduce_min_sync(0xffffffffu, lo);
                            hi = __reduce_max_sync(0xffffffffu, hi);
                            const bool none = hi == 0;           // no scale but 0, or no block: values become zeros, the scale is 0
                            int fold = none && kind == 1, general = 0;
                            if (!none && (lo != hi || __any_sync(0xffffffffu, zero != 0))) {
                                fold = !__any_sync(0xffffffffu, odd != 0) && (hi >> 23) - (lo >> 23) <= 15;
                                general = !fold;
                            }
                            if (lane == 0) {
                                mt.scale[kind] = __uint_as_float(hi);
                                mt.general[kind] = general;
                                slot.folds[kind] = fold;
                            }
                            if (fold || general) {
#pragma unroll
                                for (int i = 0; i < kTok / 32; ++i) {
                                    const int at = lane + 32 * i;
                                    float v = kind ? of[1][i] : of[0][i];
                                    if (__float_as_uint(v) == kNothing) v = 0.f;
                                    // 2^-d with d up to 15 (the last one subnormal), 0 for 0, twice in fp16
                                    const uint32_t d = (hi >> 23) - (__float_as_uint(v) >> 23);
                                    slot.fold[kind][at] = v == 0.f ? 0u : (d < 15 ? (15 - d) << 10 : 0x200u) * 0x10001u;
                                    mt.tok[kind][at] = v;
                                }
                            }
                        }
                    }
                    const int bad = slot.bad;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {    // (behind the end the limits hide the tokens)
                        const uint32_t votes = bad ? __ballot_sync(0xffffffffu, slot.block[k * 32 + lane] >= 0) : 0xffffffffu;
                        if (lane == 0) mt.valid[k] = votes;
                    }
                    if (lane == 0) mt.bad = bad;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.t_full[tile % kTileSlots]);   // (the end goes on to the loaders)
            }
        } else if (warp == 17 && lane == 0) {
            // ============================= scheduler ==============================================================
            SegmentWalk walk;
            walk.b = idle ? 0 : sm.start_b;
            walk.b_first = idle ? 0 : sm.start_units;
            walk.u = line.u0;
            for (int n = 0;; ++n) {
                wait_ring(sm, &sm.seg_empty[n % kSegments], ((n / kSegments) & 1) ^ 1, p.status);
                Segment next;
                walk.next(p, line, next);
                sm.seg[n % kSegments] = next;
                mbar_arrive(&sm.seg_full[n % kSegments]);
                if (next.n < 0) break;
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 16) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int D, int C, typename QT>
static int launch(const AttnParams& p, cudaStream_t st)
{
    constexpr size_t smem = sizeof(Shared<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory");
    auto kernel = tile_kernel<D, C, QT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) { note_cuda_error(e); (void)cudaGetLastError(); return UCMR_ERR_LAUNCH; }
    const int sms = device_sms();
    return launch_kernel(kernel, dim3(sms < kAttnMaxSms ? sms : kAttnMaxSms), dim3(kThreads), smem, st, p);
}

}  // namespace tile

template <int D>
static int tiles_typed(const AttnParams& p, int dtype, int cache_dtype, cudaStream_t st)
{
    using namespace tile;
    if (cache_dtype == UCMR_E4M3)
        return dtype == UCMR_BF16 ? launch<D, tile::kE4m3, __nv_bfloat16>(p, st) : launch<D, tile::kE4m3, __half>(p, st);
    return dtype == UCMR_BF16 ? launch<D, tile::kBf16, __nv_bfloat16>(p, st) : launch<D, tile::kF16, __half>(p, st);
}

int attention_tiles(const AttnParams& p, int D, int dtype, int cache_dtype, cudaStream_t st)
{
    return D == 64 ? tiles_typed<64>(p, dtype, cache_dtype, st) : tiles_typed<128>(p, dtype, cache_dtype, st);
}

}  // namespace ucmr
