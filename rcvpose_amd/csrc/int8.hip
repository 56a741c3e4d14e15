// int8.hip -- 8-bit integer arithmetic with one scale per token and one per output channel.
//
//   quantise  x [rows, C] (one or two channel-concatenated sources)
//             s_m = f32(max_c |x_mc| / 127),  q_mc = round-half-even(x_mc / s_m) of the exact quotient
//   product   out[m, n] = act( sw[n] * sum_tap sa[m(tap)] * (sum_k a[m(tap), k] w[n, tap, k]) + bias[n] + residual[m, n] )
//             taps = 1: rows x channels; taps = 9: a 3x3 window with zero padding over tokens that form H x W images.  The sums
//             within a tap are 32-bit integers and exact (|code| <= 128: K <= 131071 cannot overflow); the taps, whose
//             tokens have scales of their own, are added in float32 in a fixed order.
#include <math.h>

#include <algorithm>

#include "int8.hpp"

namespace rcv {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ float as_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T as_out(float v) { return (T)v; }

// round-half-even(x / s) of the exact quotient, s a normal number, |x| <= 127 s (1 + 2^-24): the product with 1/s is off by less
// than one step, and the remainder x - q s is exact in one fma (it has no more significant bits than x and s share), so comparing
// it with s / 2 settles the neighbours of a half.
__device__ __forceinline__ int quantize_exact(float x, float s, float inv)
{
    float q = rintf(x * inv);
    const float r2 = 2.f * fmaf(-q, s, x), m = fabsf(r2);
    if (m > s || (m == s && ((int)q & 1))) q += copysignf(1.f, r2);
    return (int)q;
}

template <typename T>
__global__ __launch_bounds__(256) void k_i8_quantize(const T *x0, long long pitch0, int c0, const T *x1, long long pitch1, int c1,
                                                     long long rows, int8_t *codes, long long codes_pitch, float *scales)
{
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    const int C = c0 + c1;
    float amax = 0.f, poison = 0.f;
    for (int c = lane; c < C; c += 64) {
        const float v = as_f32(c < c0 ? x0[row * pitch0 + c] : x1[row * pitch1 + c - c0]);
        amax = fmaxf(amax, fabsf(v));
        poison += v * 0.f;  // NaN once v is a NaN or an infinity
    }
    for (int o = 32; o; o >>= 1) {
        amax = fmaxf(amax, __shfl_xor(amax, o));
        poison += __shfl_xor(poison, o);
    }
    float s = __fdiv_rn(amax, 127.f);
    if (s < 0x1p-126f) s = 0.f;
    if (poison != 0.f) s = __builtin_nanf("");  // (true for a NaN only: the sum of zeros is zero)
    const float inv = s > 0.f ? 1.f / s : 0.f;
    for (int c = lane; c < C; c += 64) {
        const float v = as_f32(c < c0 ? x0[row * pitch0 + c] : x1[row * pitch1 + c - c0]);
        codes[row * codes_pitch + c] = (int8_t)(s > 0.f ? quantize_exact(v, s, inv) : 0);
    }
    if (lane == 0) scales[row] = s;
}

// v = sum * sw + bias + residual, ReLU that keeps a NaN, rounded once to the output's type
template <typename T>
__device__ __forceinline__ void i8_store(const I8Product &p, long long m, int n, float v, int g, float &vmax)
{
    v = fmaf(v, p.weight_scales[(long long)g * p.weight_scale_gs + n], p.bias ? p.bias[(long long)g * p.bias_gs + n] : 0.f);
    if (p.residual) v += as_f32(((const T *)p.residual)[(long long)g * p.residual_gs + m * p.residual_pitch + n]);
    if (p.relu) v = v < 0.f ? 0.f : v;
    vmax = fmaxf(vmax, fabsf(v));
    ((T *)p.out)[(long long)g * p.out_gs + m * p.out_pitch + n] = as_out<T>(v);
}

// 64 tokens x 64 channels per workgroup, four waves of 32 x 32, operands straight from memory.
template <typename T, int TAPS>
__global__ __launch_bounds__(256) void k_i8_simple(const I8Product p)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, kq = lane >> 4;
    const int g = blockIdx.z;
    const long long m0 = (long long)blockIdx.x * 64 + (wave >> 1) * 32;
    const int n0 = blockIdx.y * 64 + (wave & 1) * 32;
    const int8_t *codes = p.codes + (long long)g * p.code_gs * p.code_pitch;
    const float *cs = p.code_scales + (long long)g * p.code_gs;
    const int8_t *w = p.weights + (long long)g * p.Cout * TAPS * p.kp;
    f32x4 sum[2][2];
    for (int i = 0; i < 2; i++)
        for (int j = 0; j < 2; j++) sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int tap = 0; tap < TAPS; tap++) {
        long long src[2];
        for (int j = 0; j < 2; j++) {
            const long long m = m0 + j * 16 + r16;
            src[j] = m < p.rows ? m : -1;
            if (TAPS == 9 && m < p.rows) {
                const int x = (int)(m % p.W), y = (int)(m / p.W % p.H), dy = tap / 3 - 1, dx = tap % 3 - 1;
                src[j] = y + dy >= 0 && y + dy < p.H && x + dx >= 0 && x + dx < p.W ? m + (long long)dy * p.W + dx : -1;
            }
        }
        i32x4 acc[2][2];
        for (int i = 0; i < 2; i++)
            for (int j = 0; j < 2; j++) acc[i][j] = i32x4{0, 0, 0, 0};
        for (int k0 = 0; k0 < p.K; k0 += 64) {
            const int k = k0 + kq * 16;
            i32x4 wf[2], tf[2];
            for (int i = 0; i < 2; i++) {
                const int n = n0 + i * 16 + r16;
                wf[i] = n < p.Cout ? *(const i32x4 *)(w + ((long long)n * TAPS + tap) * p.kp + k) : i32x4{0, 0, 0, 0};
            }
            // (a chunk that starts below K may end behind it: inside the row's pitch, and against weights that are zero there)
            for (int j = 0; j < 2; j++)
                tf[j] = src[j] >= 0 && k < p.K ? *(const i32x4 *)(codes + src[j] * p.code_pitch + k) : i32x4{0, 0, 0, 0};
            for (int i = 0; i < 2; i++)
                for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i], tf[j], acc[i][j], 0, 0, 0);
        }
        for (int j = 0; j < 2; j++) {
            const float sa = src[j] >= 0 ? cs[src[j]] : 0.f;
            for (int i = 0; i < 2; i++)
                for (int e = 0; e < 4; e++) sum[i][j][e] = fmaf((float)acc[i][j][e], sa, sum[i][j][e]);
        }
    }
    float vmax = 0.f;
    for (int i = 0; i < 2; i++)
        for (int j = 0; j < 2; j++)
            for (int e = 0; e < 4; e++) {
                const long long m = m0 + j * 16 + r16;
                const int n = n0 + i * 16 + kq * 4 + e;
                if (m < p.rows && n < p.Cout) i8_store<T>(p, m, n, sum[i][j][e], g, vmax);
            }
    if (p.range && sizeof(T) == 2 && vmax > 65504.f) atomicOr(p.range, 2u);
}

template <typename T> int launch_quantize(const void *x0, long long pitch0, int c0, const void *x1, long long pitch1, int c1, long long rows,
                                          int8_t *codes, long long codes_pitch, float *scales, hipStream_t st)
{
    hipLaunchKernelGGL((k_i8_quantize<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, (const T *)x0, pitch0, c0, (const T *)x1,
                       pitch1, c1, rows, codes, codes_pitch, scales);
    RCV_LAUNCH_CHECK();
    return RCV_OK;
}

template <typename T> int launch_product(const I8Product &p, void *, size_t, hipStream_t st)
{
    const dim3 grid((unsigned)((p.rows + 63) / 64), (unsigned)((p.Cout + 63) / 64), p.groups);
    if (p.taps == 1) hipLaunchKernelGGL((k_i8_simple<T, 1>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_i8_simple<T, 9>), grid, dim3(256), 0, st, p);
    RCV_LAUNCH_CHECK();
    return RCV_OK;
}

}  // namespace

int i8_quantize(const void *x0, long long pitch0, int c0, const void *x1, long long pitch1, int c1, int dtype, long long rows,
                int8_t *codes, long long codes_pitch, float *scales, hipStream_t st)
{
    if (rows == 0) return RCV_OK;
    if (dtype == RCV_F32) return launch_quantize<float>(x0, pitch0, c0, x1, pitch1, c1, rows, codes, codes_pitch, scales, st);
    if (dtype == RCV_BF16) return launch_quantize<__bf16>(x0, pitch0, c0, x1, pitch1, c1, rows, codes, codes_pitch, scales, st);
    return launch_quantize<_Float16>(x0, pitch0, c0, x1, pitch1, c1, rows, codes, codes_pitch, scales, st);
}

size_t i8_product_workspace(long long, int, int, int, int) { return 0; }

int i8_product(const I8Product &p, void *ws, size_t ws_bytes, hipStream_t st)
{
    if (p.rows == 0) return RCV_OK;
    if (ws_bytes < i8_product_workspace(p.rows, p.K, p.Cout, p.taps, p.groups)) return RCV_E_WORKSPACE;
    if (p.out_dtype == RCV_F32) return launch_product<float>(p, ws, ws_bytes, st);
    if (p.out_dtype == RCV_BF16) return launch_product<__bf16>(p, ws, ws_bytes, st);
    return launch_product<_Float16>(p, ws, ws_bytes, st);
}

}  // namespace rcv

using namespace rcv;

namespace {
constexpr long long I8_MAX_ROWS = 1LL << 32;
constexpr int I8_MAX_K = 131071, I8_MAX_COUT = 1 << 20;
bool float_type(int dtype) { return dtype == RCV_F32 || dtype == RCV_BF16 || dtype == RCV_F16; }

int check_args(const rcv_i8_args *a, int taps, I8Product &p)
{
    if (!a || a->struct_bytes != sizeof(rcv_i8_args)) return RCV_E_INVALID;
    if (a->rows < 0 || a->channels <= 0 || a->out_channels <= 0) return RCV_E_INVALID;
    if (!float_type(a->out_dtype)) return RCV_E_UNSUPPORTED;
    if (a->channels > I8_MAX_K || a->out_channels > I8_MAX_COUT || a->rows > I8_MAX_ROWS) return RCV_E_TOO_LARGE;
    if (!a->codes_dev || !a->code_scales_dev || !a->weights_dev || !a->weight_scales_dev || !a->out_dev) return RCV_E_INVALID;
    if ((uintptr_t)a->codes_dev % 16 || (uintptr_t)a->weights_dev % 16 || a->codes_pitch % 16 || a->codes_pitch < a->channels)
        return RCV_E_INVALID;
    if (a->codes_pitch > (1 << 22) || a->out_pitch > (1 << 24) || (a->residual_dev && a->residual_pitch > (1 << 24))) return RCV_E_TOO_LARGE;
    const int size = a->out_dtype == RCV_F32 ? 4 : 2;
    if ((uintptr_t)a->out_dev % size || a->out_pitch < a->out_channels) return RCV_E_INVALID;
    if (a->residual_dev && ((uintptr_t)a->residual_dev % size || a->residual_pitch < a->out_channels)) return RCV_E_INVALID;
    if (taps == 9) {
        if (a->height <= 0 || a->width <= 0 || a->rows % ((long long)a->height * a->width)) return RCV_E_INVALID;
        if (a->width > (1 << 16)) return RCV_E_TOO_LARGE;
    }
    p = I8Product{};
    p.codes = a->codes_dev; p.weights = a->weights_dev;
    p.code_scales = a->code_scales_dev; p.weight_scales = a->weight_scales_dev; p.bias = a->bias_dev;
    p.residual = a->residual_dev; p.out = a->out_dev;
    p.rows = a->rows; p.code_pitch = a->codes_pitch; p.residual_pitch = a->residual_pitch; p.out_pitch = a->out_pitch;
    p.K = a->channels; p.kp = i8_kp(a->channels); p.Cout = a->out_channels; p.taps = taps;
    p.H = a->height; p.W = a->width; p.relu = a->relu != 0; p.out_dtype = a->out_dtype; p.groups = 1;
    return RCV_OK;
}
}  // namespace

extern "C" {

int rcv_i8_quantize_tokens(const void *x0_dev, long long pitch0, int c0, const void *x1_dev, long long pitch1, int c1, int dtype,
                           long long rows, int8_t *codes_dev, long long codes_pitch, float *scales_dev, void *stream)
{
    if (!x0_dev || c0 <= 0 || c1 < 0 || (c1 > 0 && !x1_dev) || rows < 0 || !codes_dev || !scales_dev) return RCV_E_INVALID;
    if (!float_type(dtype)) return RCV_E_UNSUPPORTED;
    if (c0 > I8_MAX_K || c1 > I8_MAX_K - c0 || rows > I8_MAX_ROWS) return RCV_E_TOO_LARGE;
    const int size = dtype == RCV_F32 ? 4 : 2;
    if ((uintptr_t)x0_dev % size || (uintptr_t)x1_dev % size || pitch0 < c0 || (c1 && pitch1 < c1) || codes_pitch < c0 + c1) return RCV_E_INVALID;
    if (pitch0 > (1 << 24) || (c1 && pitch1 > (1 << 24)) || codes_pitch > (1 << 24) || rows > 4LL * 0x7fffffff) return RCV_E_TOO_LARGE;
    return i8_quantize(x0_dev, pitch0, c0, x1_dev, pitch1, c1, dtype, rows, codes_dev, codes_pitch, scales_dev, (hipStream_t)stream);
}

size_t rcv_i8_matmul_workspace_bytes(long long rows, int channels, int out_channels)
{
    return rows > 0 && channels > 0 && out_channels > 0 ? i8_product_workspace(rows, channels, out_channels, 1, 1) : 0;
}

size_t rcv_i8_conv3x3_workspace_bytes(long long rows, int channels, int out_channels)
{
    return rows > 0 && channels > 0 && out_channels > 0 ? i8_product_workspace(rows, channels, out_channels, 9, 1) : 0;
}

int rcv_i8_matmul(const rcv_i8_args *args, void *ws, size_t ws_bytes, void *stream)
{
    I8Product p;
    const int rc = check_args(args, 1, p);
    return rc != RCV_OK ? rc : i8_product(p, ws, ws_bytes, (hipStream_t)stream);
}

int rcv_i8_conv3x3(const rcv_i8_args *args, void *ws, size_t ws_bytes, void *stream)
{
    I8Product p;
    const int rc = check_args(args, 9, p);
    return rc != RCV_OK ? rc : i8_product(p, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
