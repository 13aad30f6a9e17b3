// What the two attention kernels over the paged KV cache share: parameters, split of the work, per-row bookkeeping.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ucmr {

// Workspace: header (device status word first), one arrival counter per CTA, then two partial results per CTA.
constexpr int kAttnMaxCtas = 512;
constexpr int kAttnMaxRows = 16;   // query rows of a partial result
constexpr int kTileMaxCtas = 160;  // the kernel for many rows: one CTA per SM, 128 rows per partial result
constexpr size_t kAttnCounterBytes = kAttnMaxCtas * sizeof(int32_t);

inline size_t attn_workspace_bytes(int D)
{
    constexpr size_t few = (size_t)kAttnMaxCtas * 2 * kAttnMaxRows, many = (size_t)kTileMaxCtas * 2 * 128;
    return UCMR_WORKSPACE_HEADER_BYTES + kAttnCounterBytes + (few > many ? few : many) * (D + 2) * sizeof(float);
}

// Quotients by a fixed divisor (1 .. 2^31 - 1) for numbers below 2^31, without a division: n / d = (hi(m n) + n) >> l with
// l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1.
struct FastDiv {
    uint32_t m, l;
    explicit FastDiv(uint32_t d = 1)
    {
        l = 0;
        while (l < 31 && (1u << l) < d) ++l;
        m = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int div(int n) const { return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> l); }
#endif
};

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
    int32_t* counters;       // [kAttnMaxCtas], zero between launches
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

#endif

}  // namespace ucmr
