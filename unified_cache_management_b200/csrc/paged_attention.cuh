// What the two attention kernels over the paged KV cache share: parameters, split of the work, per-row bookkeeping.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ucmr {

// Workspace: header (device status word first), one arrival counter per CTA, then two partial results per CTA: at most
// kAttnPartRows rows in all, for either kernel.
constexpr int kAttnMaxSms = 152;
constexpr size_t kAttnPartRows = (size_t)kAttnMaxSms * 2 * 128;
constexpr size_t kAttnCounterBytes = 512 * sizeof(int32_t);
static_assert(kAttnCounterBytes >= 2 * kAttnMaxSms * sizeof(int32_t), "two CTAs per SM");

inline size_t attn_workspace_bytes(int D)
{
    return UCMR_WORKSPACE_HEADER_BYTES + kAttnCounterBytes + kAttnPartRows * (D + 2) * sizeof(float);
}

struct AttnParams {
    const void* q;           // [T, Hq, D]
    int64_t qs_t, qs_h;
    const void* cache[2];    // keys, values [NB, BS, Hkv, D]
    int64_t cs_b[2], cs_t[2], cs_h[2];   // strides in bytes
    const float* scale[2];   // [NB, Hkv], null for a 16-bit cache
    int64_t NB;
    int BS, Hkv, Hq, G;
    FastDiv by_block;        // division by BS
    const int32_t* table;    // [B, max_blocks] or [B, Hkv, max_blocks]
    int64_t bt_b, bt_h;
    int max_blocks;
    const int32_t* seq_lens;     // [B]
    const int32_t* query_start;  // [B + 1], null = one query token per request
    int64_t T;
    int B;
    float scale_log2;        // softmax scale * log2(e)
    int causal;
    void* out;               // [T, Hq, D]
    int64_t os_t, os_h;
    float* lse;              // [T, Hq] or null
    int32_t* status;         // first word of the workspace
    int32_t* counters;       // [CTAs], zero between launches
    float* partial;
};

#ifdef __CUDACC__

// Tokens and query tokens of a request, brought into range: a length beyond the table's blocks or a query range outside
// [0, T) would reach past the buffers.
struct AttnRequest { int len, q0, nq; };
__device__ __forceinline__ AttnRequest attn_request(const AttnParams& p, int b)
{
    AttnRequest r;
    const int64_t most = (int64_t)p.max_blocks * p.BS;
    const int len = p.seq_lens[b];
    r.len = len < 0 ? 0 : (int64_t)len > most ? (int)most : len;
    int q0 = b, q1 = b + 1;
    if (p.query_start != nullptr) { q0 = p.query_start[b]; q1 = p.query_start[b + 1]; }
    q0 = max(0, q0);
    q1 = (int)min((int64_t)q1, p.T);
    r.q0 = q0;
    r.nq = max(0, q1 - q0);
    return r;
}

// Tokens that query i of a request sees: all before and itself when causal (queries are the last tokens of the request).
__device__ __forceinline__ int attn_limit(const AttnParams& p, const AttnRequest& r, int i)
{
    return p.causal ? max(0, min(r.len, r.len - r.nq + 1 + i)) : r.len;
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> struct Out16;
template <> struct Out16<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return reinterpret_cast<const uint32_t&>(h);
    }
};
template <> struct Out16<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const __half2 h = __floats2half2_rn(a, b);
        return reinterpret_cast<const uint32_t&>(h);
    }
};

// Adds up the partial results of one item's CTAs c0 .. c1 and writes its rows.  CTA c's part lies in slot 2 c, or 2 c + 1 for
// c0, whose part is the last of its stretch; a slot holds SLOT_ROWS rows of D unnormalised values, then their references,
// then their sums.  place(row, token, head): where a row of the slot goes, false if nowhere.  A warp takes four rows at a
// time: its lanes first hold the parts' weights, then D / 32 columns each, of four parts at a time (or two).  `scratch`: WARPS * 4 *
// (D + 1) floats, so that several warps can share rows when there are few (each takes a run of the parts, and the first adds the
// others' sums up, in order).  SHARE false: a warp of its own per four rows, no barrier, and less code, where the caller's
// loops need the instruction cache (prefill of 2 x 4096 tokens: 2110 us, 2485 us with the other form).
template <int D, int SLOT_ROWS, int WARPS, bool SHARE, typename QT, typename Place>
__device__ __forceinline__ void attn_join(const AttnParams& p, int c0, int c1, int rows, int warp, int lane, float* scratch, Place place)
{
    constexpr int W = D / 32, N = 4, kFlight = SHARE ? 4 : 2;
    const float inf = __uint_as_float(0x7f800000u);
    auto slot = [&](int c) { return p.partial + ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * SLOT_ROWS * (D + 2); };
    int share = 1;                    // warps per four rows
    if constexpr (SHARE)
        while (share * 2 * ((rows + N - 1) / N) <= WARPS && share * 8 <= c1 - c0) share *= 2;
    const int which = SHARE ? warp % share : 0;
#pragma unroll 1
    for (int r0 = SHARE ? warp / share * N : warp * N; r0 < (SHARE && share > 1 ? WARPS / share * N : rows); r0 += SHARE ? WARPS / share * N : WARPS * N) {
        int64_t tok[N];
        int head[N];
        bool live[N];
        float top[N], sum[N], v[N][W];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            live[n] = r0 + n < rows && (!SHARE || place(r0 + n, tok[n], head[n]));
            top[n] = -inf;
            sum[n] = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) v[n][i] = 0.f;
        }
#pragma unroll 1
        for (int c = c0 + lane; c <= c1; c += 32)
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (live[n]) top[n] = fmaxf(top[n], __ldcg(slot(c) + SLOT_ROWS * D + r0 + n));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int n = 0; n < N; ++n) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], o));
        const int run = SHARE ? (c1 - c0 + share) / share : c1 - c0 + 1;           // parts per warp
        const int from = c0 + which * run, to = SHARE ? min(c1, from + run - 1) : c1;
#pragma unroll 1
        for (int first = from; first <= to; first += 32) {
            const int c = first + lane;
            float weight[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                weight[n] = 0.f;
                if (c <= to && live[n]) {
                    const float m = __ldcg(slot(c) + SLOT_ROWS * D + r0 + n), l = __ldcg(slot(c) + SLOT_ROWS * (D + 1) + r0 + n);
                    weight[n] = m == -inf ? 0.f : exp2_fast(m - top[n]);
                    sum[n] += m == -inf ? l : weight[n] * l;   // (a sum that is NaN stays one)
                }
            }
            const int here = min(32, to - first + 1);
#pragma unroll kFlight
            for (int k = 0; k < here; ++k) {
                const float* at = slot(first + k) + r0 * D + lane * W;
                float x[N][W];
#pragma unroll
                for (int n = 0; n < N; ++n) {
#pragma unroll
                    for (int i = 0; i < W; ++i) x[n][i] = 0.f;
                    if (!live[n]) continue;
                    if constexpr (W == 4) {
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(at + n * D));
                        x[n][0] = y.x; x[n][1] = y.y; x[n][2] = y.z; x[n][3] = y.w;
                    } else {
                        const float2 y = __ldcg(reinterpret_cast<const float2*>(at + n * D));
                        x[n][0] = y.x; x[n][1] = y.y;
                    }
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const float f = __shfl_sync(0xffffffffu, weight[n], k);
                    if (f != 0.f)
#pragma unroll
                        for (int i = 0; i < W; ++i) v[n][i] += f * x[n][i];
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int n = 0; n < N; ++n) sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], o);
        if (SHARE && share > 1) {     // (the same for the whole CTA, which comes here once)
            float* mine = scratch + warp * N * (D + 1);
#pragma unroll
            for (int n = 0; n < N; ++n) {
#pragma unroll
                for (int i = 0; i < W; ++i) mine[n * D + i * 32 + lane] = v[n][i];
                if (lane == 0) mine[N * D + n] = sum[n];
            }
            __syncthreads();
            if (which != 0) continue;
#pragma unroll 1
            for (int w = 1; w < share; ++w) {
                const float* other = mine + w * N * (D + 1);
#pragma unroll
                for (int n = 0; n < N; ++n) {
#pragma unroll
                    for (int i = 0; i < W; ++i) v[n][i] += other[n * D + i * 32 + lane];
                    sum[n] += other[N * D + n];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (!live[n] || (!SHARE && !place(r0 + n, tok[n], head[n]))) continue;
            const float inv = sum[n] == 0.f ? 0.f : 1.f / sum[n];
            QT* out = static_cast<QT*>(p.out) + tok[n] * p.os_t + (int64_t)head[n] * p.os_h + lane * W;
            if constexpr (W == 4)
                *reinterpret_cast<uint2*>(out) = make_uint2(Out16<QT>::pack(v[n][0] * inv, v[n][1] * inv), Out16<QT>::pack(v[n][2] * inv, v[n][3] * inv));
            else
                *reinterpret_cast<uint32_t*>(out) = Out16<QT>::pack(v[n][0] * inv, v[n][1] * inv);
            if (lane == 0 && p.lse != nullptr) p.lse[tok[n] * p.Hq + head[n]] = sum[n] == 0.f ? -inf : (top[n] + log2f(sum[n])) * 0.69314718055994531f;
        }
    }
}

#endif

}  // namespace ucmr
