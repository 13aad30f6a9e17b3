// Rotary positions, shared by the stand-alone rotation (rotary.cu) and the append to the paged cache (kv_append.cu).
//
// Pair i of a head is turned by the angle position * inv_freq[i].  The angle of a far position does not fit float32
// (4 Mi * 1 rad has a step of 0.25 rad), so it is counted in turns, as a 64-bit binary fraction: F = inv_freq / 2 pi
// scaled by 2^64, and position * F modulo 2^64 is the fraction of a turn - the wrap-around of the integer product IS the
// reduction.  Its top 32 bits, read as a signed number, are the angle in units of pi * 2^-31, for sincospif.  Three errors
// add up.  1 / 2 pi and its product with inv_freq are rounded to float64: off by 2^-53.3 and 2^-53 of themselves, together less
// than |position * inv_freq| * 2^-52 (inv_freq >= 0; the subtraction of whole turns is exact).  F is cut to 64 bits: at most
// |position| * 2 pi * 2^-64, which is 2^-21.3 at position 2^40.  The float32 argument: pi * 2^-25, a rounding of half a step at the
// largest argument, 1, and 2 pi * 2^-32 for the bits below the top 32, together less than 2^-23 (a 16-bit result shows no more).
// No table of cosines has to be kept or read.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ucmr {

struct RotaryAngles {
    const double* inv_freq;  // [rot / 2] radians per position; null = nothing is rotated
    const void* positions;   // [T]
    int pos_is_int64;
    int rot;                 // leading elements of a head that are rotated (even)
    int interleaved;         // pairs (2i, 2i+1) instead of (i, i + rot/2)
    float mscale;            // factor on the rotated elements
    int transpose;           // the transposed rotation (angle negated): the gradient
};

#ifdef __CUDACC__

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i)
{
    return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ float2 rotary_cos_sin(const RotaryAngles& a, int64_t position, int pair)
{
    double turns = a.inv_freq[pair] * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= floor(turns);
    const unsigned long long f = __double2ull_rz(turns * 18446744073709551616.0);  // (saturates at 2^64 - 1)
    const unsigned long long angle = f * (unsigned long long)position;
    float s, c;
    sincospif((float)(int)(angle >> 32) * 4.656612873077393e-10f /* 2^-31 */, &s, &c);
    if (a.transpose) s = -s;
    return make_float2(c * a.mscale, s * a.mscale);
}

// Two 16-bit values <-> float32.
template <typename T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
    static __device__ __forceinline__ float2 to_float(uint32_t v)
    {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t from_float(float lo, float hi)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(h);
    }
    // larger magnitudes, pair by pair, of a (not negative) and b; a NaN loses
    static __device__ __forceinline__ uint32_t abs_max(uint32_t a, uint32_t b)
    {
        const __nv_bfloat162 h = __hmax2(reinterpret_cast<const __nv_bfloat162&>(a), __habs2(reinterpret_cast<const __nv_bfloat162&>(b)));
        return reinterpret_cast<const uint32_t&>(h);
    }
    static __device__ __forceinline__ float to_float1(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_float1(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Half2<__half> {
    static __device__ __forceinline__ float2 to_float(uint32_t v) { return __half22float2(reinterpret_cast<const __half2&>(v)); }
    static __device__ __forceinline__ uint32_t from_float(float lo, float hi)
    {
        const __half2 h = __floats2half2_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(h);
    }
    static __device__ __forceinline__ uint32_t abs_max(uint32_t a, uint32_t b)
    {
        const __half2 h = __hmax2(reinterpret_cast<const __half2&>(a), __habs2(reinterpret_cast<const __half2&>(b)));
        return reinterpret_cast<const uint32_t&>(h);
    }
    static __device__ __forceinline__ float to_float1(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float1(float v) { return __float2half_rn(v); }
};

// Eight pairs of one head as two 16-byte vectors: (a[0..7], b[0..7]) with pair i = (a[i], b[i]) in the half layout,
// pairs (2i, 2i+1) running through a and then b in the interleaved one.  cs: the pairs' cosines and sines, four float4 =
// {cos, sin, cos, sin} that lie `step` apart.  x and y come back as float32 in the same order.
template <typename T>
__device__ __forceinline__ void rotate_pairs(uint4 va, uint4 vb, const float4* cs, int step, int interleaved,
                                             float (&a)[8], float (&b)[8])
{
    const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 fa = Half2<T>::to_float(wa[i]), fb = Half2<T>::to_float(wb[i]);
        a[2 * i] = fa.x; a[2 * i + 1] = fa.y;
        b[2 * i] = fb.x; b[2 * i + 1] = fb.y;
    }
    if (interleaved) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // pairs 2q, 2q+1
            const float4 t = cs[q * step];
            float* x = q < 2 ? a + 4 * q : b + 4 * (q - 2);
            const float x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
            x[0] = x0 * t.x - x1 * t.y; x[1] = x1 * t.x + x0 * t.y;
            x[2] = x2 * t.z - x3 * t.w; x[3] = x3 * t.z + x2 * t.w;
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 t = cs[q * step];
            const float a0 = a[2 * q], a1 = a[2 * q + 1], b0 = b[2 * q], b1 = b[2 * q + 1];
            a[2 * q] = a0 * t.x - b0 * t.y;     b[2 * q] = b0 * t.x + a0 * t.y;
            a[2 * q + 1] = a1 * t.z - b1 * t.w; b[2 * q + 1] = b1 * t.z + a1 * t.w;
        }
    }
}

// Where item `ch` (eight pairs) of a head starts: first vector at element `first`, second at `second`.
__device__ __forceinline__ void pair_offsets(int rot, int interleaved, int ch, int& first, int& second)
{
    first = interleaved ? ch * 16 : ch * 8;
    second = interleaved ? first + 8 : first + rot / 2;
}

// Cosines and sines of `ntok` tokens in shared memory: float4 index (token * 4 + quarter) * chunks + chunk, so that the
// threads of neighbouring chunks read neighbouring 16-byte words.
__device__ __forceinline__ void fill_cos_sin(float4* cs, const RotaryAngles& ang, int64_t pos, int row, int pair, int chunks)
{
    const int ch = pair >> 3, j = pair & 7;
    reinterpret_cast<float2*>(cs)[(((row * 4 + (j >> 1)) * chunks + ch) << 1) + (j & 1)] = rotary_cos_sin(ang, pos, pair);
}

// One rotation job: x [T, H, D] -> out, strides in elements.
struct RotaryJob {
    const void* x;
    void* out;
    int64_t T, xs_t, xs_h, os_t, os_h;
    int H, D;
    int tok_per_cta, heads_per_cta;  // tile of a CTA
    int head_tiles;
    FastDiv by_chunks, by_heads;   // divisions by the chunks per head and by heads_per_cta
};

constexpr int kRotThreads = 256;
constexpr int kRotMaxTablePairs = 4096;  // cosines and sines of a CTA's tokens: 32 KiB at most

// Tile choice: about 1024 items of eight pairs per CTA (four per thread, so that eight 16-byte loads are in flight per
// thread) once that fills the GPU twice, otherwise one item per thread, so that a decode step spreads over many SMs.
inline void plan_rotary(RotaryJob& j, int rot, int sms)
{
    const int chunks = rot / 16 > 0 ? rot / 16 : 1;
    const int64_t per_token = (int64_t)j.H * chunks;
    const int64_t items = j.T * per_token >= (int64_t)sms * 2 * 1024 ? 1024 : kRotThreads;
    if (per_token >= items) {
        j.tok_per_cta = 1;
        j.heads_per_cta = (int)(items / chunks > 0 ? items / chunks : 1);
    } else {
        int64_t t = items / per_token;
        const int64_t most = kRotMaxTablePairs / (chunks * 8) > 0 ? kRotMaxTablePairs / (chunks * 8) : 1;
        j.tok_per_cta = (int)(t < most ? t : most);
        j.heads_per_cta = j.H;
    }
    j.head_tiles = (j.H + j.heads_per_cta - 1) / j.heads_per_cta;
    j.by_chunks = FastDiv::by((uint32_t)chunks);
    j.by_heads = FastDiv::by((uint32_t)j.heads_per_cta);
}
inline int64_t rotary_ctas(const RotaryJob& j)
{
    return (j.T + j.tok_per_cta - 1) / j.tok_per_cta * j.head_tiles;
}
inline size_t rotary_smem(const RotaryJob& j, int rot) { return (size_t)j.tok_per_cta * (rot / 16) * 64; }

// The vector path reads 16-byte vectors: eight pairs per item, whole vectors behind the rotated part, aligned rows.
inline bool rotary_vector_ok(const RotaryJob& j, int rot)
{
    const uintptr_t bits = reinterpret_cast<uintptr_t>(j.x) | reinterpret_cast<uintptr_t>(j.out);
    const int64_t s = j.xs_t | j.xs_h | j.os_t | j.os_h;
    return rot % 16 == 0 && rot > 0 && j.D % 8 == 0 && bits % 16 == 0 && s % 8 == 0 && rot / 2 <= kRotMaxTablePairs;
}

// HBM-bound: each element is read and written once (2 + 2 bytes).  A CTA computes each (token, pair)'s cosine and sine
// once, in shared memory, and uses them for all its heads; the first loads are issued before that.
// 32768 tokens of 32 heads of 128: 89 us, 6.05 TB/s; a decode step's 16 tokens: 2 us in a graph.
template <typename T, int THREADS>
__device__ __forceinline__ void rotate_tile(const RotaryJob& j, const RotaryAngles& ang, int64_t cta, float4* cs)
{
    const int64_t t0 = cta / j.head_tiles * j.tok_per_cta;
    const int h0 = (int)(cta % j.head_tiles) * j.heads_per_cta;
    const int nt = (int)min((int64_t)j.tok_per_cta, j.T - t0), nh = min(j.heads_per_cta, j.H - h0);
    const int chunks = ang.rot / 16, np = ang.rot / 2;
    const int items = nt * j.heads_per_cta * chunks;
    const T* x = static_cast<const T*>(j.x) + t0 * j.xs_t + (int64_t)h0 * j.xs_h;
    T* out = static_cast<T*>(j.out) + t0 * j.os_t + (int64_t)h0 * j.os_h;
    constexpr int UN = 1024 / THREADS;
    for (int base = 0; base < items; base += 1024) {
        uint4 va[UN], vb[UN];
        int tok[UN], chn[UN], hd[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int i = base + u * THREADS + threadIdx.x, r = j.by_chunks.div(i);
            chn[u] = i - r * chunks;
            tok[u] = j.by_heads.div(r);
            hd[u] = i < items ? r - tok[u] * j.heads_per_cta : nh;   // (heads that the last tile lacks are left out)
            if (hd[u] < nh) {
                int f, s;
                pair_offsets(ang.rot, ang.interleaved, chn[u], f, s);
                const T* from = x + tok[u] * j.xs_t + hd[u] * j.xs_h;
                va[u] = *reinterpret_cast<const uint4*>(from + f);
                vb[u] = *reinterpret_cast<const uint4*>(from + s);
            }
        }
        if (base == 0) {
            for (int i = threadIdx.x; i < nt * np; i += THREADS) {
                const int row = j.by_chunks.div(i >> 3);
                fill_cos_sin(cs, ang, load_index(ang.positions, ang.pos_is_int64, t0 + row), row, i - row * np, chunks);
            }
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (hd[u] < nh) {
                float a[8], b[8];
                rotate_pairs<T>(va[u], vb[u], cs + tok[u] * 4 * chunks + chn[u], chunks, ang.interleaved, a, b);
                int f, s;
                pair_offsets(ang.rot, ang.interleaved, chn[u], f, s);
                T* o = out + tok[u] * j.os_t + hd[u] * j.os_h;
                uint4 w;
                w.x = Half2<T>::from_float(a[0], a[1]); w.y = Half2<T>::from_float(a[2], a[3]);
                w.z = Half2<T>::from_float(a[4], a[5]); w.w = Half2<T>::from_float(a[6], a[7]);
                *reinterpret_cast<uint4*>(o + f) = w;
                w.x = Half2<T>::from_float(b[0], b[1]); w.y = Half2<T>::from_float(b[2], b[3]);
                w.z = Half2<T>::from_float(b[4], b[5]); w.w = Half2<T>::from_float(b[6], b[7]);
                *reinterpret_cast<uint4*>(o + s) = w;
            }
        }
    }
    const int rest = (j.D - ang.rot) / 8;  // vectors behind the rotated part: copied, unless they are in place already
    if (rest == 0 || j.x == j.out) return;
    for (int i = threadIdx.x; i < nt * nh * rest; i += THREADS) {
        const int r = i / rest, e = ang.rot + (i - r * rest) * 8, t = r / nh, h = r - t * nh;
        *reinterpret_cast<uint4*>(out + t * j.os_t + h * j.os_h + e) = *reinterpret_cast<const uint4*>(x + t * j.xs_t + h * j.xs_h + e);
    }
}

// Any even `rot`, head size, stride and alignment: one (token, head, pair or unrotated element) per step of a thread.
template <typename T>
__device__ __forceinline__ void rotate_scalar(const RotaryJob& j, const RotaryAngles& ang, int64_t first, int64_t step)
{
    const T* x = static_cast<const T*>(j.x);
    T* out = static_cast<T*>(j.out);
    const int np = ang.rot / 2, per = np + (j.D - ang.rot);
    for (int64_t i = first; i < j.T * j.H * per; i += step) {
        const int e = (int)(i % per);
        const int64_t r = i / per;
        const int64_t t = r / j.H;
        const int h = (int)(r - t * j.H);
        const T* xr = x + t * j.xs_t + (int64_t)h * j.xs_h;
        T* orow = out + t * j.os_t + (int64_t)h * j.os_h;
        if (e >= np) {
            if (j.x != j.out) orow[e + np] = xr[e + np];
            continue;
        }
        const int ia = ang.interleaved ? 2 * e : e, ib = ang.interleaved ? 2 * e + 1 : e + np;
        const float2 cs = rotary_cos_sin(ang, load_index(ang.positions, ang.pos_is_int64, t), e);
        const float a = Half2<T>::to_float1(xr[ia]), b = Half2<T>::to_float1(xr[ib]);
        orow[ia] = Half2<T>::from_float1(a * cs.x - b * cs.y);
        orow[ib] = Half2<T>::from_float1(b * cs.x + a * cs.y);
    }
}

#endif  // __CUDACC__

}  // namespace ucmr
