// int8.hpp -- launches of the 8-bit integer operators (int8.hip) for the C ABI and for the FCN executor (fcn.hip).
#pragma once
#include "common.hpp"

namespace rcv {

// One product over all groups; a group is one network of an FCN engine (the C ABI has one group).  Group strides: tokens and weight
// rows in rows, bias and weight scales in channels (= Cout), residual and output in elements.
struct I8Product {
    const int8_t *codes, *weights;      // tokens [rows][code_pitch], weights [Cout][taps][kp]
    const float *code_scales, *weight_scales, *bias;
    const void *residual;
    void *out;
    long long rows, code_pitch, residual_pitch, out_pitch;
    long long code_gs, weight_scale_gs, bias_gs, residual_gs, out_gs;  // (the token scales' group stride is code_gs as well)
    int K, kp, Cout, taps, H, W;
    int relu, out_dtype, groups;
    bool one_order;                     // taps = 9: a window's bits do not depend on rows or groups (undivided sums)
    unsigned *range;                    // RCV_F16 engines: the sticky range-flag word, or null
};

int i8_quantize(const void *x0, long long pitch0, int c0, const void *x1, long long pitch1, int c1, int dtype, long long rows,
                int8_t *codes, long long codes_pitch, float *scales, hipStream_t st);
size_t i8_product_workspace(long long rows, int K, int Cout, int taps, int groups, bool one_order);
// No less than i8_product_workspace of these or of fewer rows.
size_t i8_product_workspace_most(long long rows, int K, int Cout, int taps, int groups, bool one_order);
int i8_product(const I8Product &p, void *ws, size_t ws_bytes, hipStream_t st);

constexpr int I8_KP = 128;  // weight rows are padded with zeros to a multiple of this many codes per tap
static inline int i8_kp(int K) { return (K + I8_KP - 1) / I8_KP * I8_KP; }

}  // namespace rcv
