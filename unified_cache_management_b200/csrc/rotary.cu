// Rotary positions (sm_100a): y = mscale * R(position * inv_freq) x on the first `rot` elements of every head, the rest
// copied.  See rotary.cuh for the angles and for the tile.  The gradient with respect to x is the transposed rotation.
#include "rotary.cuh"

namespace ucmr {

template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryJob j, const RotaryAngles ang)
{
    extern __shared__ float4 s_cs[];
    rotate_tile<T, kRotThreads>(j, ang, blockIdx.x, s_cs);
}

template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_scalar_kernel(const RotaryJob j, const RotaryAngles ang)
{
    rotate_scalar<T>(j, ang, (int64_t)blockIdx.x * kRotThreads + threadIdx.x, (int64_t)gridDim.x * kRotThreads);
}

int device_sms()
{
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

template <typename T>
static int launch_rotary(RotaryJob j, const RotaryAngles& ang, cudaStream_t st)
{
    const int sms = device_sms();
    if (rotary_vector_ok(j, ang.rot)) {
        plan_rotary(j, ang.rot, sms);
        const int64_t ctas = rotary_ctas(j);
        if (ctas > 0x7FFFFFFF) return UCMR_ERR_UNSUPPORTED;
        return launch_kernel(rotary_kernel<T>, dim3((unsigned)ctas), dim3(kRotThreads), rotary_smem(j, ang.rot), st, j, ang);
    }
    const int64_t items = j.T * j.H * (j.D - ang.rot / 2);
    const int64_t ctas = (items + kRotThreads - 1) / kRotThreads, most = (int64_t)sms * 16;
    return launch_kernel(rotary_scalar_kernel<T>, dim3((unsigned)(ctas < most ? ctas : most)), dim3(kRotThreads), 0, st, j, ang);
}

}  // namespace ucmr

extern "C" int ucmr_rotary(const void* x, void* out, int64_t T, int H, int D, int64_t x_stride_t, int64_t x_stride_h,
                           int64_t out_stride_t, int64_t out_stride_h, int dtype, const void* positions,
                           int pos_is_int64, const double* inv_freq, int rotary_dim, int interleaved, float mscale,
                           int transpose, void* stream)
{
    using namespace ucmr;
    if (T < 0 || H < 0 || D <= 0 || rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > D) return UCMR_ERR_BAD_ARG;
    if (dtype != UCMR_BF16 && dtype != UCMR_FP16) return UCMR_ERR_UNSUPPORTED;
    if (T == 0 || H == 0) return UCMR_OK;
    if (!x || !out || !positions || !inv_freq) return UCMR_ERR_BAD_ARG;
    RotaryJob j{};
    j.x = x; j.out = out; j.T = T; j.H = H; j.D = D;
    j.xs_t = x_stride_t; j.xs_h = x_stride_h; j.os_t = out_stride_t; j.os_h = out_stride_h;
    RotaryAngles a{};
    a.inv_freq = inv_freq; a.positions = positions; a.pos_is_int64 = pos_is_int64; a.rot = rotary_dim;
    a.interleaved = interleaved; a.mscale = mscale; a.transpose = transpose;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == UCMR_BF16 ? launch_rotary<__nv_bfloat16>(j, a, st) : launch_rotary<__half>(j, a, st);
}
