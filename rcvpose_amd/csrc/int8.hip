// int8.hip -- 8-bit integer arithmetic with one scale per token and one per output channel.
//
//   quantise  x [rows, C] (one or two channel-concatenated sources)
//             s_m = f32(max_c |x_mc| / 127),  q_mc = round-half-even(x_mc / s_m) of the exact quotient
//   product   out[m, n] = act( sw[n] * sum_tap sa[m(tap)] * (sum_k a[m(tap), k] w[n, tap, k]) + bias[n] + residual[m, n] )
//             taps = 1: rows x channels; taps = 9: a 3x3 window with zero padding over tokens that form H x W images.  The sums
//             within a tap are 32-bit integers and exact (|code| <= 128: K <= 131071 cannot overflow); the taps, whose
//             tokens have scales of their own, are added in float32 in an order that the sizes fix (k_i8_direct: runs of a tap's channels).
//             Float32, as nothing narrower holds the sums: it rounds the conversion, the token scale, each addition, the weight scale
//             with the bias and the residual; then the output's type rounds.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "int8.hpp"

namespace rcv {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ float as_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T as_out(float v) { return (T)v; }

// ---------------------------------------------------------------------------------------------
// quantiser
// ---------------------------------------------------------------------------------------------

// The code of x under scale s (a normal number, |x| <= 127 s (1 + 2^-24)): round-half-even(x / s) of the exact quotient in the low byte.
// `m` is x / s + MAGIC rounded, MAGIC = 1.5 * 2^23: the whole number in its low bits is off by at most one where the quotient is near a
// half.  The remainder x - q s is exact in one fma (it has no more significant bits than x and s share); a whole number gives way to its
// neighbour where twice the remainder is above s, an odd one already at s.
constexpr float MAGIC = 12582912.f;
__device__ __forceinline__ unsigned settle(float x, float s, float m)
{
    const float q = m - MAGIC, r = fmaf(-q, s, x), r2 = r + r;
    const unsigned bits = __float_as_uint(m);
    const float limit = __uint_as_float(__float_as_uint(s) - (bits & 1u));
    return bits + (fabsf(r2) > limit ? (unsigned)((__float_as_int(r2) >> 31) | 1) : 0u);
}

// The bits of |x| as a 32-bit number that orders like |x|, NaNs above the infinity.
template <typename T> __device__ __forceinline__ unsigned magnitude_bits(T v) { return __float_as_uint((float)v) & 0x7fffffffu; }

// Sixteen channels c .. c + 15 of a token, zeros behind the last.  Rows may start anywhere: the vector loads of gfx950 need no alignment.
template <typename T>
__device__ __forceinline__ void load_chunk(T *v, const T *x0, int c0, const T *x1, int C, int c)
{
    struct __attribute__((packed)) Raw { T v[16]; };
    if (c + 16 <= c0 || (c >= c0 && c + 16 <= C)) {
        const Raw r = *(const Raw *)(c < c0 ? x0 + c : x1 + (c - c0));
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = r.v[e];
    } else {
        for (int e = 0; e < 16; e++) v[e] = c + e < c0 ? x0[c + e] : c + e < C ? x1[c + e - c0] : (T)0.f;
    }
}

// The scale of a token from the largest magnitude's bits.
__device__ __forceinline__ float token_scale(unsigned bits)
{
    if (bits >= 0x7f800000u) return __builtin_nanf("");
    const float s = __fdiv_rn(__uint_as_float(bits), 127.f);
    return s < 0x1p-126f ? 0.f : s;
}

// Codes of sixteen channels.  With 1/s rounded the quotient is off by at most 127 * 2^-23 < 2^-15, so only a remainder within 2^-15 of a
// half can lead to the wrong whole number: for float32 and float16 the chunks that hold one (6 % and about 20 % of the waves) are settled
// in a second pass.  Among bfloat16's few numbers one in some hundreds is half the row's largest, whose quotient is 63.5 but for the
// rounding of s: nearly every wave would take the second pass, so each code is settled at once.
template <typename T> __device__ __forceinline__ uint4 quantize_chunk(const T *v, float s, float inv)
{
    constexpr bool AT_ONCE = std::is_same<T, __bf16>::value;
    unsigned w[4];
    float d = 0.f;
    auto put = [&](int e, unsigned bits) {
        const unsigned b = bits & 255u;
        w[e >> 2] = e & 3 ? w[e >> 2] | b << (8 * (e & 3)) : b;
    };
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float x = as_f32(v[e]), m = fmaf(x, inv, MAGIC);
        if constexpr (AT_ONCE) put(e, settle(x, s, m));
        else {
            d = fmaxf(d, fabsf(fmaf(x, inv, MAGIC - m)));
            put(e, __float_as_uint(m));
        }
    }
    if (!AT_ONCE && d > 0.5f - 0x1p-15f) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float x = as_f32(v[e]);
            put(e, settle(x, s, fmaf(x, inv, MAGIC)));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void store_chunk(int8_t *codes, uint4 w, int C, int c, bool aligned)
{
    if (aligned && c + 16 <= C) *(uint4 *)(codes + c) = w;
    else {
        const unsigned *u = (const unsigned *)&w;
        for (int e = 0; e < 16 && c + e < C; e++) codes[c + e] = (int8_t)(u[e >> 2] >> (8 * (e & 3)));
    }
}

// L lanes per token, sixteen channels a lane: one pass, the token stays in registers.  The fewest lanes that hold the token are taken, as
// idle lanes cost instructions (us, bfloat16: 100000 x 128 with 8 / 16 / 32 lanes 10.0 / 15.1 / 25.7, 300000 x 32 with 2 / 4 / 8 lanes
// 8.1 / 12.0 / 19.7, 50000 x 512 with 32 / 64 lanes 16.1 / 26.4); twice the channels in half the lanes gains nothing (100000 x 256 with 8
// lanes 17.0, 16 lanes 16.1) and lengthens small calls (300 x 1024 with 32 lanes 4.0, 64 lanes 3.4).
template <typename T, int L>
__global__ __launch_bounds__(256) void k_i8_quantize(const T *x0, long long pitch0, int c0, const T *x1, long long pitch1, int c1,
                                                     long long rows, int8_t *codes, long long codes_pitch, float *scales, bool aligned)
{
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const int lane = threadIdx.x % L, C = c0 + c1, c = lane * 16;
    if (row >= rows) return;
    T v[16];
    unsigned top = 0;
    if (c < C) load_chunk(v, x0 + row * pitch0, c0, x1 + row * pitch1, C, c);
    else
        for (int e = 0; e < 16; e++) v[e] = (T)0.f;
#pragma unroll
    for (int e = 0; e < 16; e++) top = max(top, magnitude_bits(v[e]));
#pragma unroll
    for (int o = L / 2; o; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    const float s = token_scale(top), inv = s > 0.f ? 1.f / s : 0.f;
    if (c < C) store_chunk(codes + row * codes_pitch, s > 0.f ? quantize_chunk(v, s, inv) : make_uint4(0u, 0u, 0u, 0u), C, c, aligned);
    if (lane == 0) scales[row] = s;
}

// A workgroup of NW waves per token, NV chunks of sixteen channels a lane in registers.  NV = 0: a token of any length, read twice (the
// second time from the caches).
// Bound by memory: 63600 tokens of 2048 channels, in bfloat16 75 us and in float16 67 us (391 MB: 5.2 and 5.9 TB/s, a copy reaches 5.1), in
// float32 115 us (652 MB: 5.7 TB/s).  A single token of 4096 channels: 3 us.  Shapes, us for bfloat16 / float16 / float32: 63600 x 2048 with 128
// lanes of one chunk 75 / 67 / 115, 64 of two 73 / 71 / 119, and a single token 3.1 / 2.8 / 2.8 against 3.7 / 3.3 / 3.3; 30000 x 4096 with
// 256 of one 68 / 65 / 107, 128 of two 69 / 68 / 112, 64 of four 75 / 70 / 114; 10000 x 5000 with 256 of two 32 / 29 / 40, 512 of one
// 36 / 34 / 38; 8192 x 16384 with 1024 of one 77 / 72 / 117, read twice 90 / 83 / 150.
template <typename T, int NW, int NV>
__global__ __launch_bounds__(64 * NW) void k_i8_quantize_wide(const T *x0, long long pitch0, int c0, const T *x1, long long pitch1, int c1,
                                                              int8_t *codes, long long codes_pitch, float *scales, bool aligned)
{
    constexpr int LANES = 64 * NW;
    __shared__ unsigned tops[NW];
    const long long row = blockIdx.x;
    const int C = c0 + c1, first = threadIdx.x * 16;
    const T *t0 = x0 + row * pitch0, *t1 = x1 + row * pitch1;
    T v[NV ? NV : 1][16];
    unsigned top = 0;
    auto scan = [&](const T *u) {
#pragma unroll
        for (int e = 0; e < 16; e++) top = max(top, magnitude_bits(u[e]));
    };
    if constexpr (NV == 0) {
        for (int c = first; c < C; c += LANES * 16) {
            load_chunk(v[0], t0, c0, t1, C, c);
            scan(v[0]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = i * LANES * 16 + first;
            if (c < C) load_chunk(v[i], t0, c0, t1, C, c);
            else
                for (int e = 0; e < 16; e++) v[i][e] = (T)0.f;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) scan(v[i]);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) top = max(top, tops[w]);
    const float s = token_scale(top), inv = s > 0.f ? 1.f / s : 0.f;
    auto store = [&](const T *u, int c) {
        store_chunk(codes + row * codes_pitch, s > 0.f ? quantize_chunk(u, s, inv) : make_uint4(0u, 0u, 0u, 0u), C, c, aligned);
    };
    if constexpr (NV == 0) {
        for (int c = first; c < C; c += LANES * 16) {
            load_chunk(v[0], t0, c0, t1, C, c);
            store(v[0], c);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (i * LANES * 16 + first < C) store(v[i], i * LANES * 16 + first);
    }
    if (threadIdx.x == 0) scales[row] = s;
}

// A view of memory for buffer loads: what lies beyond `bytes` reads as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t view(const int8_t *base, long long bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes < 0 ? 0 : bytes > 0x7fffffffLL ? 0x7fffffff : (int)bytes, 0x00020000);
}
__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t rsrc, int voff, int soff)
{
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, voff, soff, 0));
}

// N consecutive channels of a row that may start anywhere (gfx950's vector accesses need no alignment)
template <typename T, int N> struct Row {
    typedef T Vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N> __device__ __forceinline__ typename Row<T, N>::Vec load_row(const T *x, int n, int Cout)
{
    typename Row<T, N>::Vec r = {};
    if (n + N <= Cout) r = *(const typename Row<T, N>::Vec *)x;
    else
        for (int e = 0; e < N; e++) if (n + e < Cout) r[e] = x[e];
    return r;
}
template <typename T> __device__ __forceinline__ const T *residual_row(const I8Product &p, int g, long long m)
{
    return p.residual ? (const T *)p.residual + (long long)g * p.residual_gs + m * p.residual_pitch : nullptr;
}
// Channels n .. n + N - 1 of token m, scaled and with the bias: residual, ReLU that keeps a NaN, rounded once to the output's type.  Returns
// the largest magnitude stored.
template <typename T, int N>
__device__ __forceinline__ float finish_row(const I8Product &p, int g, long long m, int n, float *v, typename Row<T, N>::Vec res)
{
    T *out = (T *)p.out + (long long)g * p.out_gs + m * p.out_pitch + n;
    float vmax = 0.f;
    typename Row<T, N>::Vec o;
#pragma unroll
    for (int e = 0; e < N; e++) {
        if (p.residual) v[e] += as_f32(res[e]);
        if (p.relu) v[e] = v[e] < 0.f ? 0.f : v[e];
        if (n + e < p.Cout) vmax = fmaxf(vmax, fabsf(v[e]));
        o[e] = as_out<T>(v[e]);
    }
    if (n + N <= p.Cout) *(typename Row<T, N>::Vec *)out = o;
    else
        for (int e = 0; e < N; e++) if (n + e < p.Cout) out[e] = o[e];
    return vmax;
}
// Four channels whose sums still lack the weight scales and the bias.
template <typename T> __device__ __forceinline__ float finish_quad(const I8Product &p, int g, long long m, int n, const float *sum)
{
    const float *ws = p.weight_scales + (long long)g * p.weight_scale_gs + n, *bias = p.bias ? p.bias + (long long)g * p.bias_gs + n : nullptr;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const bool live = n + e < p.Cout;
        v[e] = fmaf(sum[e], live ? ws[e] : 0.f, live && bias ? bias[e] : 0.f);
    }
    const T *res = residual_row<T>(p, g, m);
    return finish_row<T, 4>(p, g, m, n, v, res ? load_row<T, 4>(res + n, n, p.Cout) : typename Row<T, 4>::Vec{});
}
template <typename T> __device__ __forceinline__ void report_range(const I8Product &p, float vmax)
{
    if (sizeof(T) == 2 && p.range && vmax > 65504.f) atomicOr(p.range, 2u);
}

// ---------------------------------------------------------------------------------------------
// operands straight from memory: few output tiles
// ---------------------------------------------------------------------------------------------

// TT * 16 tokens x CT * 16 channels per workgroup.  Its NW waves -- and the workgroups of gridDim.y -- divide the sum among themselves:
// every wave multiplies its own run of 64-channel steps with nothing shared, D steps of loads in flight, so a short call is a few
// memory round trips long.  The waves' sums meet in LDS and are added in order; with gridDim.y > 1 they go to `partial`
// [split][group][rows][quads] and k_i8_finish adds them in order.  Integer sums (TAPS = 1) are exact whatever the order.
// Bound by memory where one token meets many weights (1 x 8192 -> 32768: 268 MB in 43 us, 6.2 TB/s), by the depth of the loads in flight
// where there is little to read (300 x 2048 -> 512: 7.8 us, of which a launch is 2.8).  Two workgroups on a CU count for more than deeper
// loads: windows of 64 tokens with D = 1 in 96 registers against D = 2 in 136, 3 x 37 x 53, 96 -> 80 8.8 / 10.9 us.
template <typename T, int TAPS, int TT, int CT, int NW, int D>
__global__ __launch_bounds__(64 * NW, CT == 1 ? 4 : 2) void k_i8_direct(const I8Product p, int tiles_n, f32x4 *partial)
{
    constexpr int OOB = (int)0x80000000, TILE_N = CT * 16, ROW = TILE_N + 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kq = lane >> 4;
    const int g = blockIdx.z, mt = blockIdx.x / tiles_n, nt = blockIdx.x - mt * tiles_n, n0 = nt * TILE_N;
    const long long m0 = (long long)mt * (TT * 16);
    const int left = (int)min((long long)(TT * 16), p.rows - m0);
    const int8_t *codes = p.codes + (long long)g * p.code_gs * p.code_pitch;
    const int8_t *codes_end = codes + (p.rows - 1) * p.code_pitch + ((p.K + 15) & ~15);
    const float *cs = p.code_scales + (long long)g * p.code_gs;
    const int wrow = TAPS * p.kp, W = p.W, H = p.H;
    const int8_t *wts = p.weights + ((long long)g * p.Cout + n0) * wrow;
    const long long wbytes = (long long)(p.Cout - n0) * wrow;

    int toff[TT], woff[CT];
    unsigned inside[TT];
#pragma unroll
    for (int j = 0; j < TT; j++) {
        const int row = j * 16 + r16;
        toff[j] = row < left ? (int)(row * p.code_pitch) + kq * 16 : OOB;
        inside[j] = 0u;
        if (TAPS == 9 && row < left) {
            const long long m = m0 + row, l = m / W;
            const int x = (int)(m - l * W), y = (int)(l % H);
            const unsigned cols = (x > 0 ? 1u : 0u) | 2u | (x + 1 < W ? 4u : 0u);
            inside[j] = (y > 0 ? cols : 0u) | cols << 3 | (y + 1 < H ? cols << 6 : 0u);
        }
    }
#pragma unroll
    for (int i = 0; i < CT; i++) woff[i] = (i * 16 + r16) * wrow + kq * 16;

    const int ksteps = (p.K + 63) / 64, nk = TAPS * ksteps;
    const int unit = blockIdx.y * NW + wave, units = gridDim.y * NW;
    const int s0 = (int)((long long)nk * unit / units), s1 = (int)((long long)nk * (unit + 1) / units);
    int tap = TAPS == 9 ? s0 / ksteps : 0, ks = s0 - tap * ksteps;  // of the step being loaded
    auto tap_shift = [&](int t) { return TAPS == 9 ? (long long)(t / 3 - 1) * W + (t % 3 - 1) : 0LL; };
    auto load = [&](i32x4 *tf, i32x4 *wf, int step) {
        if (step >= s1) return;
        const int8_t *a = codes + (m0 + tap_shift(tap)) * p.code_pitch, *w = wts + (long long)tap * p.kp;
        const __amdgpu_buffer_rsrc_t ra = view(a, codes_end - a), rw = view(w, wbytes - (long long)tap * p.kp);
#pragma unroll
        for (int i = 0; i < CT; i++) wf[i] = load16(rw, woff[i], ks * 64);
#pragma unroll
        for (int j = 0; j < TT; j++) tf[j] = load16(ra, TAPS == 1 || (inside[j] >> tap) & 1u ? toff[j] : OOB, ks * 64);
        if (++ks == ksteps) { ks = 0; tap++; }
    };

    i32x4 acc[CT][TT], tf[2][D][TT], wf[2][D][CT];
    f32x4 sum[CT][TT];
#pragma unroll
    for (int i = 0; i < CT; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) {
            acc[i][j] = i32x4{0, 0, 0, 0};
            sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    int m_tap = TAPS == 9 ? s0 / ksteps : 0, m_ks = s0 - m_tap * ksteps;  // of the step being multiplied
    auto step_of = [&](const i32x4 *t, const i32x4 *w, int step) {
        if (step >= s1) return;
#pragma unroll
        for (int i = 0; i < CT; i++)
#pragma unroll
            for (int j = 0; j < TT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], t[j], acc[i][j], 0, 0, 0);
        if (TAPS == 9 && (++m_ks == ksteps || step + 1 == s1)) {  // the tokens of the next tap have scales of their own
#pragma unroll
            for (int j = 0; j < TT; j++) {
                const float sa = (inside[j] >> m_tap) & 1u ? cs[m0 + j * 16 + r16 + tap_shift(m_tap)] : 0.f;
#pragma unroll
                for (int i = 0; i < CT; i++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) sum[i][j][e] = fmaf((float)acc[i][j][e], sa, sum[i][j][e]);
                    acc[i][j] = i32x4{0, 0, 0, 0};
                }
            }
            m_ks = 0;
            m_tap++;
        }
    };
#pragma unroll
    for (int d = 0; d < D; d++) load(tf[0][d], wf[0][d], s0 + d);
    for (int s = s0; s < s1; s += 2 * D) {
#pragma unroll
        for (int f = 0; f < 2; f++) {
#pragma unroll
            for (int d = 0; d < D; d++) load(tf[1 - f][d], wf[1 - f][d], s + (f + 1) * D + d);
#pragma unroll
            for (int d = 0; d < D; d++) step_of(tf[f][d], wf[f][d], s + f * D + d);
        }
    }

    // the waves' sums meet: [wave][token][channel]
#pragma unroll
    for (int i = 0; i < CT; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) {
            const int at = ((wave * TT + j) * 16 + r16) * ROW + i * 16 + kq * 4;
            if constexpr (TAPS == 9) ((f32x4 *)smem)[at / 4] = sum[i][j];
            else ((i32x4 *)smem)[at / 4] = acc[i][j];
        }
    __syncthreads();
    float vmax = 0.f;
    for (int q = tid; q < TT * 16 * CT * 4; q += 64 * NW) {
        const int row = q / (CT * 4), n = n0 + (q - row * (CT * 4)) * 4;
        if (row >= left || n >= p.Cout) continue;
        const int at = row * (ROW / 4) + (q - row * (CT * 4));
        f32x4 v;
        if constexpr (TAPS == 9) {
            v = ((const f32x4 *)smem)[at];
#pragma unroll
            for (int w = 1; w < NW; w++) {
                const f32x4 o = ((const f32x4 *)smem)[at + w * TT * 16 * (ROW / 4)];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += o[e];
            }
        } else {
            i32x4 t = ((const i32x4 *)smem)[at];
#pragma unroll
            for (int w = 1; w < NW; w++) t += ((const i32x4 *)smem)[at + w * TT * 16 * (ROW / 4)];
            v = __builtin_bit_cast(f32x4, t);
        }
        if (partial) {
            const long long quads = (p.Cout + 3) / 4;
            partial[(((long long)blockIdx.y * p.groups + g) * p.rows + m0 + row) * quads + n / 4] = v;
            continue;
        }
        if constexpr (TAPS == 1) {
            const i32x4 t = __builtin_bit_cast(i32x4, v);
            const float sa = cs[m0 + row];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = (float)t[e] * sa;
        }
        vmax = fmaxf(vmax, finish_quad<T>(p, g, m0 + row, n, (const float *)&v));
    }
    report_range<T>(p, vmax);
}

// Adds the partial sums of a divided product in order and finishes.
template <typename T, int TAPS> __global__ __launch_bounds__(256) void k_i8_finish(const I8Product p, const f32x4 *partial, int splits)
{
    const int quads = (p.Cout + 3) / 4, g = blockIdx.z;
    const long long q = (long long)blockIdx.x * 256 + threadIdx.x;
    if (q >= p.rows * quads) return;
    const long long m = q / quads, stride = (long long)p.groups * p.rows * quads;
    const f32x4 *at = partial + (long long)g * p.rows * quads + q;
    f32x4 v = at[0];
    constexpr int AHEAD = 8;  // parts requested together
    for (int s0 = 1; s0 < splits; s0 += AHEAD) {
        f32x4 o[AHEAD];
#pragma unroll
        for (int s = 0; s < AHEAD; s++) o[s] = s0 + s < splits ? at[(s0 + s) * stride] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < AHEAD; s++) {
            if (s0 + s >= splits) continue;
            if constexpr (TAPS == 9) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += o[s][e];
            } else
                v = __builtin_bit_cast(f32x4, __builtin_bit_cast(i32x4, v) + __builtin_bit_cast(i32x4, o[s]));
        }
    }
    if constexpr (TAPS == 1) {
        const i32x4 t = __builtin_bit_cast(i32x4, v);
        const float sa = p.code_scales[(long long)g * p.code_gs + m];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (float)t[e] * sa;
    }
    report_range<T>(p, finish_quad<T>(p, g, m, (int)(q - m * quads) * 4, (const float *)&v));
}

// ---------------------------------------------------------------------------------------------
// operands through LDS
// ---------------------------------------------------------------------------------------------

// One piece of an operand tile: 64 lanes x 16 bytes from `at` + soff + voff to LDS bytes [lds + LDS_OFF, + 1024).  Lanes whose offset (soff
// included) is not below `bytes` deliver zeros.
struct View {
    long long at;
    int bytes;
};
template <int LDS_OFF> __device__ __forceinline__ void dma16(const View &v, int soff, unsigned lds, int voff)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)v.at, 0, v.bytes, 0x00020000),
                                             (__attribute__((address_space(3))) void *)(uintptr_t)(lds + LDS_OFF), 16, voff, soff, 0, 0);
}
// All but the newest N pieces of every wave have landed, and all LDS reads before are done.  (The compiler does not wait for the pieces: it
// does not connect them with the reads.  It moves no access to memory past either statement.)
template <int N> __device__ __forceinline__ void step_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int I, int N, typename F> __device__ __forceinline__ void for_each(F &&f)  // f(I) ... f(N - 1), each a compile-time constant
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        for_each<I + 1, N>(f);
    }
}

// r[i] of the four 16-lane rows k <-> r[k] of row i: a 4 x 4 transposition between registers and rows of lanes.
__device__ __forceinline__ void transpose_rows(float &r0, float &r1, float &r2, float &r3)
{
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    auto swap32 = [](float &a, float &b) {  // the upper half of a <-> the lower half of b
        const u32x2 v = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        a = __uint_as_float(v[0]);
        b = __uint_as_float(v[1]);
    };
    auto swap16 = [](float &a, float &b) {  // the odd rows of a <-> the even rows of b
        const u32x2 v = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        a = __uint_as_float(v[0]);
        b = __uint_as_float(v[1]);
    };
    swap32(r0, r2);
    swap32(r1, r3);
    swap16(r0, r1);
    swap16(r2, r3);
}

template <int TAPS_, int WT_, int WC_, int TT_, int CT_, int NA_, int NB_, bool SPLIT_ = false> struct TileShape {
    static constexpr bool SPLIT = SPLIT_;  // the sum may be divided over workgroups
    static constexpr int TAPS = TAPS_, WT = WT_, WC = WC_, TT = TT_, CT = CT_, NA = NA_, NB = NB_;
    static constexpr int KB = 128;                                // codes of a row per step: one cache line
    static constexpr int NW = WT * WC, BM = WT * TT * 16, BN = WC * CT * 16;
    static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;      // pieces (8 rows) of a wave per step
    static constexpr int A_BYTES = BM * KB, B_BYTES = BN * KB, B_RING = NA * A_BYTES, TABLE = B_RING + NB * B_BYTES;
    static constexpr int LDS = TABLE + (TAPS == 9 ? 9 * BM * 4 : 0);
    static constexpr bool STAGED = TT * CT <= 8;                  // the epilogue goes through LDS
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && LDS <= 160 * 1024 && NA >= 3 && NB >= 2 && NB <= NA && BM <= 64 * NW && CT == 4, "tile plan");
    // Pieces in order of issue, per step kt: the tokens of step kt + NA - 1 in its first half, the weights of step kt + NB in its second.
    // Half-way through step kt everything of step kt + 1 has to be there: what may still be on its way was issued later.
    static constexpr int LATE = NB == NA ? (NA - 2) * (PA + PB) : (NB - 2) * (PA + PB) + PA;
};

// BM tokens x BN channels per workgroup, WT x WC waves of TT x CT 16 x 16 tiles.  The weights are the matrix instruction's first operand, so a
// lane ends up with four consecutive channels of one token.  Rings of NA token and NB weight stages of 128 codes a row; the eight 16-byte
// chunks of a row are permuted (chunk ^= row bits) on the way in, so that the sixteen rows of a fragment read fall on all banks.
// One barrier per step, half-way: before it a wave has read the step's last fragments, behind it the next step's first are there.
//
// TAPS = 9 walks tap by tap.  The integer sums of a tap are scaled into `sum` between the first products of the next.
//
// What bounds it: at long sums the card's power (16384 x 8192 -> 8192: 828 us, 2.66 POP/s, matrix units 0.66 busy at 1.7 to 1.8 GHz; a loop
// of the same instructions on registers 3.4 to 3.95) and, for windows, the copies into LDS (53 x 30 x 40, 2048 -> 512: 502 us, 2.4
// POP/s; without its products 377 us, without its copies 339).  At short ones a tile's start and end: 2 and 5 us beside 0.7 us a step (24 x
// 120 x 160, 512 -> 128: 314 us, 1.7 POP/s).  Fewer bytes per product are what helps, hence tiles as large as the registers allow.
//
// gridDim.y > 1 divides the sum: a workgroup takes its share of the channels (TAPS = 1) or of the taps and leaves raw sums in `partial`
// [split][group][rows][quads of channels] for k_i8_finish.
template <typename T, typename S>
__global__ __launch_bounds__(64 * S::NW, 2) void k_i8_tile(const I8Product p, int tiles_m, int tiles_n, f32x4 *partial)
{
    constexpr int TAPS = S::TAPS, TT = S::TT, CT = S::CT, KB = S::KB, PA = S::PA, PB = S::PB, BM = S::BM, BN = S::BN;
    constexpr int OOB = (int)0x80000000;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wave / S::WC, wc = wave % S::WC, r16 = lane & 15, kq = lane >> 4;

    // Workgroups go round-robin over the 8 XCDs: give every XCD a contiguous run of tiles, and walk a run in bands of eight
    // token tiles, so that the tiles in flight on an XCD share both operands in its L2.
    int mt, nt;
    {
        const unsigned total = gridDim.x, id = blockIdx.x, q = total / 8, r = total % 8, xcd = id % 8;
        const unsigned s = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + id / 8;
        const unsigned band = 8u * tiles_n, bi = s / band, in = s - bi * band;
        const unsigned rows = min(8u, (unsigned)tiles_m - bi * 8);
        nt = __builtin_amdgcn_readfirstlane((int)(in / rows));
        mt = __builtin_amdgcn_readfirstlane((int)(bi * 8 + in % rows));
    }
    const int g = blockIdx.z, n0 = nt * BN;
    const long long m0 = (long long)mt * BM;
    const int left = (int)min((long long)BM, p.rows - m0);
    const int8_t *codes = p.codes + (long long)g * p.code_gs * p.code_pitch;
    const float *cs = p.code_scales + (long long)g * p.code_gs;
    const int wrow = TAPS * p.kp;
    const int8_t *wts = p.weights + ((long long)g * p.Cout + n0) * wrow;

    // which of the nine taps of a token lie inside its image
    const int W = p.W, H = p.H;
    int x0 = 0, y0 = 0;
    const float rw = 1.f / (float)max(W, 1), rh = 1.f / (float)max(H, 1);
    if constexpr (TAPS == 9) {
        const long long l = m0 / W;
        x0 = __builtin_amdgcn_readfirstlane((int)(m0 - l * W));
        y0 = __builtin_amdgcn_readfirstlane((int)(l % H));
    }
    auto taps_inside = [&](int row) -> unsigned {
        if (row >= left) return 0u;
        // The image row l rows below the tile's first.  (A product with the reciprocal, half a step up: the quotient is at most BM for W = 1 and 1
        // for the widest image of 65536 columns, its error far below the half step's distance 1 / (2 W) to a whole number.)
        const int t = x0 + row, l = (int)(((float)t + 0.5f) * rw), x = t - l * W, yl = y0 + l;
        // Heights have no such bound (float32 misplaces the last row of 6556022), but the tile reaches fewer than BM rows down: a taller image
        // ends in it at most once, and for a lower one yl < 2 BM.
        const int y = yl - (H >= BM ? (yl >= H ? H : 0) : (int)(((float)yl + 0.5f) * rh) * H);
        const unsigned cols = (x > 0 ? 1u : 0u) | 2u | (x + 1 < W ? 4u : 0u);
        return (y > 0 ? cols : 0u) | cols << 3 | (y + 1 < H ? cols << 6 : 0u);
    };
    // What a staged epilogue needs, requested first: the scales of this lane's tokens, the scales and biases of the V channels it will finish.
    constexpr int V = 16 / sizeof(T), CPR = BN / V;
    const int c = tid % CPR, n = n0 + c * V;
    float sa[TT] = {};
    typename Row<float, V>::Vec sw = {}, bias = {};
    auto load_token_scales = [&]() {
#pragma unroll
        for (int j = 0; j < TT; j++) {
            const int row = (wt * TT + j) * 16 + r16;
            sa[j] = row < left ? cs[m0 + row] : 0.f;
        }
    };
    if constexpr (S::STAGED && !S::SPLIT) {
        if constexpr (TAPS == 1) load_token_scales();
        sw = load_row<float, V>(p.weight_scales + (long long)g * p.weight_scale_gs + n, n, p.Cout);
        if (p.bias) bias = load_row<float, V>(p.bias + (long long)g * p.bias_gs + n, n, p.Cout);
    }

    // this lane's part of the pieces: row lane / 8 of the piece, 16-byte slot lane % 8
    auto chunk_of = [&](int row, int slot) { return slot ^ ((row >> 1) & 7); };
    int aoff[PA], boff[PB];
    unsigned inside[TAPS == 9 ? PA : 1];
#pragma unroll
    for (int c = 0; c < PA; c++) {
        const int row = (wave * PA + c) * 8 + lane / 8;
        aoff[c] = row < left ? (int)(row * p.code_pitch) + chunk_of(row, lane % 8) * 16 : OOB;
        if constexpr (TAPS == 9) inside[c] = taps_inside(row);
    }
#pragma unroll
    for (int c = 0; c < PB; c++) {
        const int row = (wave * PB + c) * 8 + lane / 8;
        boff[c] = row * wrow + chunk_of(row, lane % 8) * 16;
    }

    // Where the next token and the next weight pieces come from.  Behind the last step the pieces go on with every lane out of range, which
    // keeps the counts the same.
    const long long pitch = p.code_pitch;
    const int units = TAPS == 9 ? 9 : (p.K + KB - 1) / KB;  // what a split takes a run of
    const int u0 = S::SPLIT ? (int)(units * blockIdx.y / gridDim.y) : 0, u1 = S::SPLIT ? (int)(units * (blockIdx.y + 1) / gridDim.y) : units;
    const int tap0 = TAPS == 9 ? u0 : 0, tap1 = TAPS == 9 ? u1 : 1;
    const int klo = TAPS == 9 ? 0 : u0 * KB, khi = TAPS == 9 ? (p.K + KB - 1) / KB * KB : u1 * KB;
    struct Walk { int tap, k, done; };
    auto step = [&](Walk &w) -> bool {  // true where another tap begins
        w.k += KB;
        if (w.k < khi) return false;
        w.k = klo;
        if constexpr (TAPS == 9) {
            w.tap++;
            if (w.tap < tap1) return true;
            w.tap = tap0;
        }
        w.done = OOB;
        return false;
    };
    Walk ia{tap0, klo, 0}, ib{tap0, klo, 0};
    unsigned a_lds = lds0 + wave * PA * 1024, b_lds = lds0 + S::B_RING + wave * PB * 1024;
    const unsigned a_last = a_lds + (S::NA - 1) * S::A_BYTES, b_last = b_lds + (S::NB - 1) * S::B_BYTES;
    // The descriptors of a tap, in few scalar instructions (every wave runs them, all matrix units wait): the tokens move by `shift` rows, and
    // the view ends with the tile's or the tensor's last row, whichever comes first.
    View ra, rb;
    const long long next_col = pitch, next_row = (long long)(W - 2) * pitch;
    const int below = (int)min(p.rows - m0, 1LL << 30), last_row = (int)pitch - ((p.K + 15) & ~15);
    long long a_at = (long long)(codes + (m0 + (TAPS == 9 ? (long long)(tap0 / 3 - 1) * W + (tap0 % 3 - 1) : 0)) * pitch);
    int a_col = tap0 % 3, shift = TAPS == 9 ? (tap0 / 3 - 1) * W + a_col - 1 : 0;
    long long b_at = (long long)(wts + (long long)tap0 * p.kp);
    int b_bytes = min(p.Cout - n0, BN) * wrow - tap0 * p.kp;
    auto a_view = [&]() {
        const int rows = min(below - shift, BM);
        ra = View{a_at, rows > 0 ? rows * (int)pitch - last_row : 0};
    };
    auto b_view = [&]() { rb = View{b_at, b_bytes}; };
    auto a_tap = [&]() {
        const bool wrap = ++a_col == 3;
        a_col = wrap ? 0 : a_col;
        a_at += wrap ? next_row : next_col;
        shift += wrap ? W - 2 : 1;
        a_view();
    };
    auto b_tap = [&]() {
        b_at += p.kp;
        b_bytes -= p.kp;
        b_view();
    };
    auto a_piece = [&](auto cc) {
        constexpr int c = decltype(cc)::value;
        int v = aoff[c];
        if constexpr (TAPS == 9) v = (inside[c] >> ia.tap) & 1u ? v : OOB;
        dma16<c * 1024>(ra, ia.k, a_lds, v | ia.done);
    };
    auto b_piece = [&](auto cc) {
        constexpr int c = decltype(cc)::value;
        dma16<c * 1024>(rb, ib.k, b_lds, boff[c] | ib.done);
    };
    auto a_end = [&]() {
        a_lds = a_lds == a_last ? a_last - (S::NA - 1) * S::A_BYTES : a_lds + S::A_BYTES;
        if (step(ia)) a_tap();
    };
    auto b_end = [&]() {
        b_lds = b_lds == b_last ? b_last - (S::NB - 1) * S::B_BYTES : b_lds + S::B_BYTES;
        if (step(ib)) b_tap();
    };

    // [9][BM] in LDS: the scale under which a token's tap enters, 0 outside the image (there the offset is out of range and the load gives 0).
    // Requested before the pieces, so that storing them waits for no piece.
    float tap_scale[9] = {};
    if constexpr (TAPS == 9) {
        const __amdgpu_buffer_rsrc_t view_s = view((const int8_t *)(cs + (m0 - W - 1)), (p.rows - m0 + W + 1) * 4);
        const unsigned ok = tid < BM ? taps_inside(tid) : 0u;
#pragma unroll
        for (int t = 0; t < 9; t++)
            tap_scale[t] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(view_s, (ok >> t) & 1u ? (tid + (t / 3) * W + t % 3) * 4 : OOB, 0, 0));
    }
    a_view();
    b_view();
#pragma unroll
    for (int s = 0; s < S::NA - 1; s++) {  // tokens of steps 0 .. NA - 2 and weights of steps 0 .. NB - 1 in the order of the loop
        for_each<0, PA>(a_piece);
        a_end();
        if (s >= S::NA - 1 - S::NB) {
            for_each<0, PB>(b_piece);
            b_end();
        }
    }
    if constexpr (S::NB == S::NA) {
        for_each<0, PB>(b_piece);
        b_end();
    }

    float *sa_tab = (float *)(smem + S::TABLE);
    if constexpr (TAPS == 9)
        if (tid < BM) {
#pragma unroll
            for (int t = 0; t < 9; t++) sa_tab[t * BM + tid] = tap_scale[t];
        }

    i32x4 acc[CT][TT];
    f32x4 sum[TAPS == 9 ? CT : 1][TAPS == 9 ? TT : 1];
#pragma unroll
    for (int i = 0; i < CT; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) {
            acc[i][j] = i32x4{0, 0, 0, 0};
            if constexpr (TAPS == 9) sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    float sc[TT] = {};  // TAPS = 9: the scales of the tap whose sums are in acc
    i32x4 tf[2][TT], wf[2][CT];
    const int t_row = (wt * TT * 16 + r16) * KB, w_row = S::B_RING + (wc * CT * 16 + r16) * KB;
    int a_stage = 0, b_stage = 0;  // byte offsets of the stages being read
    auto read = [&](int f, int half, int q) {  // fragment q of set f
        const int slot = chunk_of(r16, half * 4 + kq) * 16;
        if (q < TT) tf[f][q] = *(const i32x4 *)(smem + a_stage + t_row + slot + q * 16 * KB);
        else wf[f][q - TT] = *(const i32x4 *)(smem + b_stage + w_row + slot + (q - TT) * 16 * KB);
    };
    // all products of fragment set f; meanwhile the other set is read from `half` of the current stages and N pieces are issued
    constexpr int NM = TT * CT, NF = TT + CT, SEG = NM / 4, RSEG = SEG / 2;  // (the reads go into the first half: they are back before the barrier)
    auto multiply = [&](auto ff, int half, auto count, auto &&piece, auto first) {
        constexpr int f = decltype(ff)::value, n = decltype(count)::value;
        for_each<0, SEG>([&](auto ss) {
            constexpr int s = decltype(ss)::value;
#pragma unroll
            for (int q = 0; q < NF; q++) if (q * RSEG / NF == s) read(1 - f, half, q);
            for_each<s * n / SEG, (s + 1) * n / SEG>(piece);
            if constexpr (decltype(first)::value) {
#pragma unroll
                for (int e = s * 4; e < s * 4 + 4; e++) {
                    const int i = e / TT, j = e % TT;
#pragma unroll
                    for (int q = 0; q < 4; q++) sum[i][j][q] = fmaf((float)acc[i][j][q], sc[j], sum[i][j][q]);
                    asm volatile("" : "+v"(sum[i][j]));  // (here: put off, it would keep the old sums in registers of their own)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[f][i], tf[f][j], i32x4{0, 0, 0, 0}, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                // (reads, half of the products, a piece, the others: with its addresses computed under the first two products a piece costs
                // less than in the compiler's order: 518 against 526 us for the window over 53 images of 30 x 40, 2048 -> 512 channels)
                __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
#pragma unroll
                for (int e = s * 4; e < s * 4 + 4; e++) {
                    const int i = e / TT, j = e % TT;
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[f][i], tf[f][j], acc[i][j], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    constexpr std::integral_constant<int, 0> c0{};
    constexpr std::integral_constant<int, 1> c1{};
    constexpr std::integral_constant<int, PA> pa{};
    constexpr std::integral_constant<int, PB> pb{};

    step_barrier<S::LATE + PB>();
#pragma unroll
    for (int q = 0; q < NF; q++) read(0, 0, q);
    auto finish_step = [&]() {
        a_end();
        step_barrier<S::LATE>();  // the next step is here; nobody reads the current one any more
        a_stage = a_stage == (S::NA - 1) * S::A_BYTES ? 0 : a_stage + S::A_BYTES;
        b_stage = b_stage == (S::NB - 1) * S::B_BYTES ? 0 : b_stage + S::B_BYTES;
        multiply(c1, 0, pb, b_piece, std::false_type{});
        b_end();
    };
    for (int tap = tap0; tap < tap1; tap++) {
        int k = klo;
        if constexpr (TAPS == 9) {
            multiply(c0, 1, pa, a_piece, std::true_type{});
#pragma unroll
            for (int j = 0; j < TT; j++) sc[j] = sa_tab[tap * BM + wt * TT * 16 + j * 16 + r16];
            finish_step();
            k += KB;
        }
        for (; k < khi; k += KB) {
            multiply(c0, 1, pa, a_piece, std::false_type{});
            finish_step();
        }
    }
    if constexpr (TAPS == 9) {
#pragma unroll
        for (int i = 0; i < CT; i++)
#pragma unroll
            for (int j = 0; j < TT; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) sum[i][j][q] = fmaf((float)acc[i][j][q], sc[j], sum[i][j][q]);
    }
    float vmax = 0.f;
    if constexpr (S::STAGED) {
        // The scaled sums go through LDS, so that rows leave (and the residual's rows come) in whole lines.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // (the last pieces: zeros nobody reads)
        constexpr int SROW = BN + 4, ROUND = 64 * S::NW / CPR;
        static_assert(BM * SROW * 4 <= S::LDS, "the tile fits");
        float *stage = (float *)smem;
        __syncthreads();  // the rings have been read
#pragma unroll
        for (int i = 0; i < CT; i++) {
            const int col = (wc * CT + i) * 16 + kq * 4;
#pragma unroll
            for (int j = 0; j < TT; j++) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (TAPS == 9) v[e] = sum[i][j][e];
                    else v[e] = S::SPLIT ? __int_as_float(acc[i][j][e]) : (float)acc[i][j][e] * sa[j];
                }
                *(f32x4 *)(stage + ((wt * TT + j) * 16 + r16) * SROW + col) = v;
            }
        }
        __syncthreads();
        constexpr int AHEAD = 4;  // residual rows requested together
        static_assert(BM % (ROUND * AHEAD) == 0, "whole rounds");
        if constexpr (S::SPLIT) {  // raw sums: float32 (TAPS = 9) or integers
            const long long quads = (p.Cout + 3) / 4;
            for (int row = tid / (BN / 4); row < BM; row += 64 * S::NW / (BN / 4)) {
                const int col = tid % (BN / 4);
                if (row < left && n0 + col * 4 < p.Cout)
                    partial[(((long long)blockIdx.y * p.groups + g) * p.rows + m0 + row) * quads + n0 / 4 + col] = *(const f32x4 *)(stage + row * SROW + col * 4);
            }
        } else if (n < p.Cout)
            for (int r0 = tid / CPR; r0 < BM; r0 += ROUND * AHEAD) {
                typename Row<T, V>::Vec res[AHEAD] = {};
                if (p.residual) {
#pragma unroll
                    for (int a = 0; a < AHEAD; a++) {
                        const int row = r0 + a * ROUND;
                        if (row < left) res[a] = load_row<T, V>(residual_row<T>(p, g, m0 + row) + n, n, p.Cout);
                    }
                }
#pragma unroll
                for (int a = 0; a < AHEAD; a++) {
                    const int row = r0 + a * ROUND;
                    if (row >= left) continue;
                    float v[V];
#pragma unroll
                    for (int q = 0; q < V / 4; q++) *(f32x4 *)(v + 4 * q) = *(const f32x4 *)(stage + row * SROW + c * V + 4 * q);
#pragma unroll
                    for (int e = 0; e < V; e++) v[e] = fmaf(v[e], sw[e], bias[e]);
                    vmax = fmaxf(vmax, finish_row<T, V>(p, g, m0 + row, n, v, res[a]));
                }
            }
    } else {
        // Every wave finishes its part from registers.  A lane takes N consecutive channels of a token: 16-bit rows leave as whole 128-byte lines
        // after a 4 x 4 transposition between a lane's four tiles and the four rows of lanes, float32 rows as 64-byte pieces of their own.
        // (Against the way through LDS: 16384 x 1024 -> 4096 108 -> 101 us, the window over 53 images of 30 x 40, 2048 -> 512 channels 499 ->
        // 492 us; the small tiles lose by it, 16384 x 256 -> 2048 30.2 -> 31.3 us.)
        constexpr int N = sizeof(T) == 2 ? 16 : 4, Q = 16 / N;
        auto channel = [&](int q) { return n0 + wc * CT * 16 + (N == 16 ? kq * 16 : q * 16 + kq * 4); };
        typename Row<float, N>::Vec ws[Q] = {}, bs[Q] = {};
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int nq = channel(q);
            if (nq < p.Cout) {
                ws[q] = load_row<float, N>(p.weight_scales + (long long)g * p.weight_scale_gs + nq, nq, p.Cout);
                if (p.bias) bs[q] = load_row<float, N>(p.bias + (long long)g * p.bias_gs + nq, nq, p.Cout);
            }
        }
        if constexpr (TAPS == 1) load_token_scales();
        constexpr int AHEAD = 4;  // residual rows requested together
        static_assert(TT % AHEAD == 0, "whole rounds");
#pragma unroll
        for (int j0 = 0; j0 < TT; j0 += AHEAD) {
            typename Row<T, N>::Vec res[AHEAD][Q] = {};
            if (p.residual) {
#pragma unroll
                for (int a = 0; a < AHEAD; a++) {
                    const int row = (wt * TT + j0 + a) * 16 + r16;
#pragma unroll
                    for (int q = 0; q < Q; q++) {
                        const int nq = channel(q);
                        if (row < left && nq < p.Cout) res[a][q] = load_row<T, N>(residual_row<T>(p, g, m0 + row) + nq, nq, p.Cout);
                    }
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                const int j = j0 + a, row = (wt * TT + j) * 16 + r16;
                float v[CT][4];
#pragma unroll
                for (int i = 0; i < CT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (TAPS == 9) v[i][e] = sum[i][j][e];
                        else v[i][e] = (float)acc[i][j][e] * sa[j];
                    }
                if constexpr (N == 16) {
#pragma unroll
                    for (int e = 0; e < 4; e++) transpose_rows(v[0][e], v[1][e], v[2][e], v[3][e]);
                }
#pragma unroll
                for (int q = 0; q < Q; q++) {
                    const int nq = channel(q);
                    if (row >= left || nq >= p.Cout) continue;
                    float o[N];
#pragma unroll
                    for (int e = 0; e < N; e++) o[e] = fmaf(v[q + e / 4][e % 4], ws[q][e], bs[q][e]);
                    vmax = fmaxf(vmax, finish_row<T, N>(p, g, m0 + row, nq, o, res[a][q]));
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // (the last pieces: zeros nobody reads)
    }
    report_range<T>(p, vmax);
}

template <typename T>
int launch_quantize(const void *x0_, long long pitch0, int c0, const void *x1_, long long pitch1, int c1, long long rows, int8_t *codes,
                    long long codes_pitch, float *scales, hipStream_t st)
{
    const T *x0 = (const T *)x0_, *x1 = (const T *)x1_;
    const int C = c0 + c1;
    const bool aligned = (uintptr_t)codes % 16 == 0 && codes_pitch % 16 == 0;
    // a launch holds fewer than 2^32 threads: `per` tokens at most
    auto in_parts = [&](long long per, auto &&launch) -> int {
        for (long long r = 0; r < rows; r += per) {
            launch(x0 + r * pitch0, x1 ? x1 + r * pitch1 : x1, std::min(per, rows - r), codes + r * codes_pitch, scales + r);
            RCV_LAUNCH_CHECK();
        }
        return RCV_OK;
    };
#define RCV_I8_Q(L)                                                                                                               \
    if (C <= L * 16)                                                                                                              \
        return in_parts((1LL << 31) / L, [&](const T *a, const T *b, long long n, int8_t *q, float *s) {                          \
            hipLaunchKernelGGL((k_i8_quantize<T, L>), dim3((unsigned)((n + 256 / L - 1) / (256 / L))), dim3(256), 0, st, a, pitch0, c0, b, \
                               pitch1, c1, n, q, codes_pitch, s, aligned);                                                        \
        });
    RCV_I8_Q(1)
    RCV_I8_Q(2)
    RCV_I8_Q(4)
    RCV_I8_Q(8)
    RCV_I8_Q(16)
    RCV_I8_Q(32)
    RCV_I8_Q(64)
#undef RCV_I8_Q
#define RCV_I8_Q(NW, NV)                                                                                                          \
    if (!NV || C <= 64 * NW * NV * 16)                                                                                             \
        return in_parts((1LL << 31) / (64 * NW), [&](const T *a, const T *b, long long n, int8_t *q, float *s) {                  \
            hipLaunchKernelGGL((k_i8_quantize_wide<T, NW, NV>), dim3((unsigned)n), dim3(64 * NW), 0, st, a, pitch0, c0, b, pitch1, c1, q, \
                               codes_pitch, s, aligned);                                                                          \
        });
    RCV_I8_Q(2, 1)
    RCV_I8_Q(4, 1)
    RCV_I8_Q(4, 2)
    RCV_I8_Q(16, 1)
    RCV_I8_Q(16, 0)
#undef RCV_I8_Q
    return RCV_E_TOO_LARGE;
}

// Lets `kernel` use more than the default 64 KB of LDS on the current device, once (ready: one bit per device).
int allow_lds(const void *kernel, int bytes, std::atomic<unsigned long long> &ready)
{
    int dev = 0;
    RCV_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 64 && ready.load(std::memory_order_acquire) >> dev & 1) return RCV_OK;
    RCV_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 64) ready.fetch_or(1ULL << dev, std::memory_order_release);
    return RCV_OK;
}

// How a product runs.
struct Plan {
    enum Kind { WIDE /* SQUARE for short sums: wide_from */, TALL, SQUARE, NARROW, DIRECT } kind;
    int splits;
    size_t bytes;  // of partial sums
    bool wide_direct;  // DIRECT: two 16-channel tiles a workgroup
};

// The times beside the rules are microseconds of one call in a graph, bfloat16 out; M x K -> N for a product, images x height x width, K -> N
// for a window.
Plan plan_product(long long rows, int K, int Cout, int taps, int groups, bool one_order)
{
    Plan pl{Plan::SQUARE, 1, 0, false};
    // k_i8_tile adds the nine taps one after the other, whatever its tiles; k_i8_direct and divided sums scale and add other pieces of them.
    const bool whole = one_order && taps == 9;
    const int steps = taps * ((K + 127) / 128);
    auto tiles = [&](int bm, int bn) { return ((rows + bm - 1) / bm) * ((Cout + bn - 1) / bn) * groups; };

    // Straight from memory, where the tiles are few and read few bytes of tokens (each reads its own: with all weights read once, 4 x 8192 ->
    // 32768 takes 45, through LDS 50; 8 rows 51 / 51, 16 rows 64 / 54).  Direct / through LDS: 300 x 2048 -> 512 7.8 / 10.5,
    // 128 x 1024 -> 1024 5.4 / 8.0, 32 x 4096 -> 4096 9.0 / 11.2, 64 x 4096 -> 4096 12.9 / 12.4, 64 x 8192 -> 8192 26 / 20; more than 64
    // rows: 512 x 1024 -> 1024 8.3 / 8.1, 1000 x 2048 -> 1000 17 / 12, short sums 391 x 291 -> 1136 4.9 / 7.1, 603 x 532 -> 1994 10.6 / 8.3;
    // windows: 3 x 37 x 53, 96 -> 80 8.8 / 13.1, 1 x 60 x 80, 64 -> 64 7.6 / 12.9, 64 -> 128 11.2 / 12.5, 128 -> 128 18.1 / 12.5,
    // 1 x 13 x 58, 168 -> 467 9.7 / 14.2, 1 x 15 x 20, 1024 -> 256 17.2 / 13.2, 1 x 30 x 40, 512 -> 128 14.8 / 13.2.
    const long long small = tiles(64, 16);
    // (two 16-channel tiles per workgroup share the tokens once all CUs are busy: 32 x 1024 -> 8192 5.2 / 6.1, 64 x 2048 -> 8192 9.8 / 12.5,
    // but 32 x 4096 -> 4096 10.6 / 8.9)
    pl.wide_direct = taps == 1 && rows > 16 && small >= 512;
    const double token_bytes = (double)(pl.wide_direct ? tiles(64, 32) : small) * std::min(rows, 64LL) * taps * ((K + 63) & ~63);
    const bool few = small <= 320 || (small <= 640 && (taps == 9 || token_bytes <= 16000000));
    // (windows whose rows lie whole cache lines apart read few of the cache's channels at a time: 1 x 30 x 40, 256 -> 256 15.2 / 14.0, but
    // 3 x 21 x 18, 355 -> 208 9.7 / 14.4)
    if (!whole && (rows <= 4 || (token_bytes <= (taps == 9 && K % 128 == 0 ? 42000000 : 60000000) && (rows <= 64 || few)))) {
        pl.kind = Plan::DIRECT;
        // Workgroups divide a long sum while CUs are free.  In 1 / 2 / 4 / 8 parts: 1 x 16384 -> 512 11.7 / 9.4 / 7.7 / 7.5, 1 x 4096 -> 512
        // 5.3 / 6.1 / 6.2 / 7.0, 1 x 8192 -> 64 7.3 / 7.0 / 6.8, 45 x 2343 -> 758 5.9 / 7.1, 64 x 4096 -> 512 12.0 / 9.9 / 8.4; windows
        // 1 x 8 x 8, 2048 -> 256 39 / 24 / 17 / 14, 1 x 5 x 7, 512 -> 64 10.7 / 10.1 / 8.9 / 9.2, 1 x 20 x 5, 369 -> 112 11.2 / 10.9 / 9.3,
        // 1 x 17 x 4, 288 -> 645 8.3 / 9.0, 3 x 26 x 8, 147 -> 30 7.0 / 8.2.
        const int steps64 = taps * ((K + 63) / 64);
        const int least = taps == 9 ? 54 : rows > 16 ? 47 : 128, part = taps == 9 ? 13 : rows > 32 ? 16 : rows > 16 ? 24 : 32;
        if (steps64 >= least)
            while (pl.splits < 8 && small * pl.splits * 2 <= 256 && steps64 >= pl.splits * 2 * part) pl.splits *= 2;
    } else {
        // rounds of the chip's 256 CUs times the relative time of a tile
        auto cost = [&](int bm, int bn, double w) { return (double)((tiles(bm, bn) + 255) / 256) * w; };
        if (taps == 1) {
            // 256 x 256 tiles move half the bytes of 128 x 128 ones, but need full rounds, and a long sum behind their start and end
            // (wide_from).  256 / 128: 3328 x 4096 -> 4096 (rounds filled to 0.81) 55 / 64, 2816 rows (0.69) 51 / 52, 4608 rows (0.56)
            // 98 / 81, 2048 rows (0.50) 49 / 36.
            const long long wide = tiles(256, 256);
            if (wide * 4 >= 3 * ((wide + 255) / 256 * 256)) pl.kind = Plan::WIDE;
        } else if (Cout <= 64) {
            // 256 x 64 tiles against 128 x 128 ones that are half empty: 16 x 240 x 320, 192 -> 64 336 / 618, 3 x 120 x 160, 256 -> 64 19 / 33;
            // where each needs one round the times are equal (1 x 120 x 160 17.2 / 17.1) and the smaller tiles can be divided by taps.
            if (cost(256, 64, 0.66) <= cost(128, 128, 0.62)) pl.kind = Plan::NARROW;
        } else if (cost(256, 128, 1.0) <= cost(128, 128, 0.62))
            // 256 x 128 / 128 x 128: 53 x 30 x 40, 2048 -> 512 551 / 663, 8 x 60 x 80, 128 -> 128 20 / 25; one round of either:
            // 12 x 15 x 20, 2048 -> 1024 106 / 83
            pl.kind = Plan::TALL;
        if (pl.kind == Plan::SQUARE && !whole) {
            // Few tiles of a long sum: workgroups divide it while the CUs hold them at once.  In 1 / 3 / 9 parts (taps): 1 x 15 x 20,
            // 2048 -> 1024 67 / 30 / 23, 1 x 30 x 40, 2048 -> 512 68 / 32 / 33, 3 x 28 x 43, 717 -> 127 30 / 19 / 24, 1 x 60 x 80,
            // 1024 -> 256 39 / 27 / 44, 512 -> 256 23 / 24 / 35, 128 -> 256 13 / 21 / 37, 2 x 69 x 54, 488 -> 61 24 / 17 / 28,
            // 3 x 29 x 33, 313 -> 452 20 / 30 / 38, 1 x 30 x 40, 512 -> 512 23 / 18 / 26, 256 -> 512 16 / 16 / 26; in 1 / 2 / 4 parts
            // (channels): 697 x 2907 -> 493 14.2 / 13.2 / 12.6, 512 x 8192 -> 1024 35 / 21 / 17, 512 x 8192 -> 2048 35 / 24 / 27,
            // 1024 x 8192 -> 2048 37 / 34 / 44, 64 x 4096 -> 4096 16 / 13 / 12, 512 x 4096 -> 2048 17 / 20 / 20.
            const long long wgs = tiles(128, 128);
            if (taps == 9) pl.splits = wgs <= 24 && steps >= 36 ? 9 : wgs <= 85 && steps >= (wgs <= 48 ? 18 : 27) ? 3 : 1;
            else if (steps >= (wgs <= 40 ? 20 : 48))
                while (wgs * pl.splits * 2 <= (pl.splits == 1 ? 256 : 160) && steps >= pl.splits * 2 * 8) pl.splits *= 2;
        }
    }
    if (pl.splits > 1) pl.bytes = (size_t)pl.splits * groups * rows * ((Cout + 3) / 4) * 16;
    return pl;
}

template <typename T, int TAPS> int launch_finish(const I8Product &p, const Plan &pl, const void *partial, hipStream_t st)
{
    const long long quads = p.rows * ((p.Cout + 3) / 4);
    hipLaunchKernelGGL((k_i8_finish<T, TAPS>), dim3((unsigned)((quads + 255) / 256), 1, p.groups), dim3(256), 0, st, p, (const f32x4 *)partial,
                       pl.splits);
    RCV_LAUNCH_CHECK();
    return RCV_OK;
}

template <typename T, typename S> int launch_tile(const I8Product &p, const Plan &pl, void *ws, hipStream_t st)
{
    const long long tm = (p.rows + S::BM - 1) / S::BM, tn = (p.Cout + S::BN - 1) / S::BN;
    if (tm * tn * 64 * S::NW > 0xffffffffLL) return RCV_E_TOO_LARGE;  // (threads of a launch)
    static std::atomic<unsigned long long> ready{0};
    const int rc = allow_lds((const void *)k_i8_tile<T, S>, S::LDS, ready);
    if (rc != RCV_OK) return rc;
    f32x4 *partial = S::SPLIT ? (f32x4 *)ws : nullptr;
    hipLaunchKernelGGL((k_i8_tile<T, S>), dim3((unsigned)(tm * tn), pl.splits, p.groups), dim3(64 * S::NW), S::LDS, st, p, (int)tm, (int)tn, partial);
    RCV_LAUNCH_CHECK();
    return partial ? launch_finish<T, S::TAPS>(p, pl, partial, st) : RCV_OK;
}

template <typename T, int TAPS, int TT, int CT, int D> int launch_direct(const I8Product &p, const Plan &pl, void *ws, hipStream_t st)
{
    constexpr int NW = 8, LDS = NW * TT * 16 * (CT * 16 + 4) * 4;
    static std::atomic<unsigned long long> ready{0};
    if (LDS > 64 * 1024) {
        const int rc = allow_lds((const void *)k_i8_direct<T, TAPS, TT, CT, NW, D>, LDS, ready);
        if (rc != RCV_OK) return rc;
    }
    const long long tm = (p.rows + TT * 16 - 1) / (TT * 16), tn = (p.Cout + CT * 16 - 1) / (CT * 16);
    f32x4 *partial = pl.splits > 1 ? (f32x4 *)ws : nullptr;
    hipLaunchKernelGGL((k_i8_direct<T, TAPS, TT, CT, NW, D>), dim3((unsigned)(tm * tn), pl.splits, p.groups), dim3(64 * NW), LDS, st, p, (int)tn,
                       partial);
    RCV_LAUNCH_CHECK();
    return partial ? launch_finish<T, TAPS>(p, pl, partial, st) : RCV_OK;
}

// The shortest sum for which 256 x 256 tiles pay.  256 / 128, us, 16384 rows -> 4096 channels: bfloat16, 512 69 / 71, 768 81 / 86, 1024 91 / 99,
// 2048 135 / 153, 8192 400 / 483; with a residual 768 113 / 121, 2560 192 / 203; float32 768 108 / 100, 1536 144 / 139, 2560 194 / 194, 4096
// 261 / 278 (in one round, 4096 rows: 768 32 / 32, 2560 51 / 56).  They finish from registers, with less to hide it behind, and some ends
// need a longer sum to pay for them, each about as much again:
// - 16-bit rows that start anywhere.  4001 channels: 1536 143 / 130, 2048 163 / 154, 2560 188 / 185, 3328 219 / 226; 4096 rows: 2048 47 / 46,
//   2560 53 / 54.
// - residuals in pieces of lines.  bfloat16, 4008 channels: 2048 183 / 175, 2560 207 / 204, 3328 236 / 243.  float32 crosses by the rounds
//   that are behind each other: 4 (16384 rows) 2048 246 / 216, 2560 275 / 255, 3328 302 / 302, 4096 337 / 339; 2 (8192 rows) 2048 125 / 126,
//   2560 139 / 142; 1 (4096 rows) 1024 44 / 47, 2560 64 / 69; 4001 channels in 4 rounds 2048 246 / 228, 2560 271 / 268, 3328 302 / 309.
// - both: 4001 channels of bfloat16 3328 266 / 247, 4096 294 / 291, 4608 318 / 319; 4096 rows 4096 78 / 77, 4608 84 / 84.
template <typename T> int wide_from(const I8Product &p)
{
    const long long pitch = p.out_pitch * (long long)sizeof(T);
    return 768 + (sizeof(T) == 2 && pitch % 16 ? 1792 : 0) + (p.residual && (sizeof(T) == 4 || pitch % 128) ? 1792 : 0);
}

template <typename T, int TAPS> int launch_taps(const I8Product &p, const Plan &pl, void *ws, hipStream_t st)
{
    if (pl.kind == Plan::DIRECT) {
        if (p.rows <= 16) return launch_direct<T, TAPS, 1, 1, TAPS == 1 ? 4 : 2>(p, pl, ws, st);
        if constexpr (TAPS == 1)
            if (pl.wide_direct) return p.rows <= 32 ? launch_direct<T, 1, 2, 2, 2>(p, pl, ws, st) : launch_direct<T, 1, 4, 2, 2>(p, pl, ws, st);
        if (p.rows <= 32) return launch_direct<T, TAPS, 2, 1, TAPS == 1 ? 4 : 2>(p, pl, ws, st);
        return launch_direct<T, TAPS, 4, 1, TAPS == 1 ? 2 : 1>(p, pl, ws, st);
    }
    if constexpr (TAPS == 1) {
        if (pl.kind == Plan::WIDE && p.K >= wide_from<T>(p)) return launch_tile<T, TileShape<1, 2, 4, 8, 4, 3, 2>>(p, pl, ws, st);
        if (pl.splits > 1) return launch_tile<T, TileShape<1, 4, 2, 2, 4, 5, 4, true>>(p, pl, ws, st);
        return launch_tile<T, TileShape<1, 4, 2, 2, 4, 3, 2>>(p, pl, ws, st);
    } else {
        if (pl.kind == Plan::TALL) return launch_tile<T, TileShape<9, 4, 2, 4, 4, 3, 3>>(p, pl, ws, st);
        if (pl.kind == Plan::NARROW) return launch_tile<T, TileShape<9, 8, 1, 2, 4, 3, 3>>(p, pl, ws, st);
        if (pl.splits > 1) return launch_tile<T, TileShape<9, 4, 2, 2, 4, 5, 4, true>>(p, pl, ws, st);
        return launch_tile<T, TileShape<9, 4, 2, 2, 4, 5, 4>>(p, pl, ws, st);
    }
}

template <typename T> int launch_product(const I8Product &p, void *ws, hipStream_t st)
{
    const Plan pl = plan_product(p.rows, p.K, p.Cout, p.taps, p.groups, p.one_order);
    return p.taps == 9 ? launch_taps<T, 9>(p, pl, ws, st) : launch_taps<T, 1>(p, pl, ws, st);
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

size_t i8_product_workspace(long long rows, int K, int Cout, int taps, int groups, bool one_order)
{
    return rows > 0 ? plan_product(rows, K, Cout, taps, groups, one_order).bytes : 0;
}

// plan_product divides a sum while its tiles (of at most 128 x 128) times its parts are at most 256, by channels into eight parts or parts of
// at least eight steps, by taps into nine.
size_t i8_product_workspace_most(long long rows, int K, int Cout, int taps, int groups, bool one_order)
{
    constexpr long long ALL = 256 * 128 * 128 * 4;
    if (rows <= 0 || (taps == 9 && one_order)) return 0;
    const long long parts = taps == 9 ? 9 : std::max(8, (K + 127) / 128 / 8), row = parts * groups * ((Cout + 3) / 4) * 16;
    return (size_t)(rows > ALL / row ? ALL : rows * row);
}

int i8_product(const I8Product &p, void *ws, size_t ws_bytes, hipStream_t st)
{
    if (p.rows == 0) return RCV_OK;
    const size_t need = i8_product_workspace(p.rows, p.K, p.Cout, p.taps, p.groups, p.one_order);
    if (need && (ws_bytes < need || !ws)) return RCV_E_WORKSPACE;
    if ((uintptr_t)ws % 16) return RCV_E_INVALID;
    if (p.out_dtype == RCV_F32) return launch_product<float>(p, ws, st);
    if (p.out_dtype == RCV_BF16) return launch_product<__bf16>(p, ws, st);
    return launch_product<_Float16>(p, ws, st);
}

}  // namespace rcv

using namespace rcv;

namespace {
constexpr long long I8_MAX_ROWS = 1LL << 32;
constexpr int I8_MAX_K = 131071, I8_MAX_COUT = 1 << 20;
// Sizes that check_args takes: what plan_product computes of them stays within its integers.
bool countable(long long rows, int channels, int out_channels)
{
    return rows > 0 && rows <= I8_MAX_ROWS && channels > 0 && channels <= I8_MAX_K && out_channels > 0 && out_channels <= I8_MAX_COUT;
}
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
    if ((uintptr_t)a->code_scales_dev % 4 || (uintptr_t)a->weight_scales_dev % 4 || (uintptr_t)a->bias_dev % 4) return RCV_E_INVALID;
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
    if ((uintptr_t)scales_dev % 4) return RCV_E_INVALID;
    if ((uintptr_t)x0_dev % size || (uintptr_t)x1_dev % size || pitch0 < c0 || (c1 && pitch1 < c1) || codes_pitch < c0 + c1) return RCV_E_INVALID;
    if (pitch0 > (1 << 24) || (c1 && pitch1 > (1 << 24)) || codes_pitch > (1 << 24) || rows > 0x7fffffff) return RCV_E_TOO_LARGE;
    return i8_quantize(x0_dev, pitch0, c0, x1_dev, pitch1, c1, dtype, rows, codes_dev, codes_pitch, scales_dev, (hipStream_t)stream);
}

size_t rcv_i8_matmul_workspace_bytes(long long rows, int channels, int out_channels)
{
    return countable(rows, channels, out_channels) ? i8_product_workspace(rows, channels, out_channels, 1, 1, false) : 0;
}

size_t rcv_i8_conv3x3_workspace_bytes(long long rows, int channels, int out_channels)
{
    return countable(rows, channels, out_channels) ? i8_product_workspace(rows, channels, out_channels, 9, 1, false) : 0;
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
