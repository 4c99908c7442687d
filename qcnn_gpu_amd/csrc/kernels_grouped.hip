// Products grouped by expert (qcnn_op_grouped_matmul).
#include "block_ops.h"

namespace qcnn {

template <typename T> struct Acc { typedef float type; };
template <> struct Acc<int8_t> { typedef int type; };
__device__ __forceinline__ int to_acc(int8_t v) { return v; }
template <typename T> __device__ __forceinline__ float to_acc(T v) { return to_f32(v); }

template <typename T>
__global__ __launch_bounds__(256) void k_grouped_simple(const qcnn_grouped_matmul_t a)
{
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (size_t)a.rows * a.n) return;
    const int r = (int)(at / a.n), j = (int)(at % a.n);
    int e = 0;
    while (e < a.experts && !(a.offsets[e] <= r && r < a.offsets[e + 1])) ++e;
    if (e == a.experts) return;
    const int src = a.src ? a.src[r] : r;
    const bool have = src >= 0 && src < a.x_rows;
    const T *x = (const T *)a.x + (size_t)src * a.ldx;
    const T *w = (const T *)a.w + (size_t)e * a.w_stride + (size_t)j * a.ldw;
    typename Acc<T>::type acc = 0;
    if (have)
        for (int k = 0; k < a.k; ++k) acc += to_acc(w[k]) * to_acc(x[k]);
    float v = (float)acc;
    if (a.w_scale) v *= a.w_scale[(size_t)e * a.n + j];
    if (a.x_scale && have) v *= a.x_scale[src];
    if (a.bias) v += a.bias[(size_t)e * a.n + j];
    v = block_act(v, a.act);
    if (a.row_scale) v *= a.row_scale[r];
    store_typed(a.y, (size_t)r * a.ldy + j, a.out_type, v);
}

hipError_t launch_grouped_matmul(const qcnn_grouped_matmul_t &a, hipStream_t s)
{
    const unsigned blocks = (unsigned)(((size_t)a.rows * a.n + 255) / 256);
    if (a.type == QCNN_F32)
        k_grouped_simple<float><<<blocks, 256, 0, s>>>(a);
    else if (a.type == QCNN_F16)
        k_grouped_simple<f16_t><<<blocks, 256, 0, s>>>(a);
    else if (a.type == QCNN_BF16)
        k_grouped_simple<bf16_t><<<blocks, 256, 0, s>>>(a);
    else
        k_grouped_simple<int8_t><<<blocks, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace qcnn
