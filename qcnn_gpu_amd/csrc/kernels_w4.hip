// Products with 4-bit weights and group scales (qcnn_op_matvec_w4).
#include "block_ops.h"

namespace qcnn {

template <typename T>
__global__ __launch_bounds__(256) void k_w4_simple(const qcnn_matvec_w4_t a)
{
    const size_t at = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // one wave an output
    if (at >= (size_t)a.rows * a.n) return;
    const int m = (int)(at / a.n), j = (int)(at % a.n), lane = threadIdx.x & 63;
    const T *x = (const T *)a.x + (size_t)m * a.ldx;
    const uint8_t *w = (const uint8_t *)a.w + (size_t)j * a.ldw;
    float acc = 0.f;
    for (int k = lane; k < a.k; k += 64) {
        const size_t g = (size_t)(k / a.group) * a.n + j;
        const int q = (w[k >> 1] >> ((k & 1) * 4)) & 15;
        const int z = a.zero ? ((const uint8_t *)a.zero)[g] : 8;
        acc += (float)(q - z) * load_typed(a.scale, g, a.scale_type) * to_f32(x[k]);
    }
    for (int o = 32; o; o >>= 1) acc += __shfl_xor(acc, o);
    if (lane == 0) store_typed(a.y, (size_t)m * a.ldy + j, a.out_type, a.bias ? acc + ((const float *)a.bias)[j] : acc);
}

hipError_t launch_matvec_w4(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    const size_t blocks = ((size_t)a.rows * a.n + 3) / 4;
    if (a.type == QCNN_F32)
        k_w4_simple<float><<<(unsigned)blocks, 256, 0, s>>>(a);
    else if (a.type == QCNN_F16)
        k_w4_simple<f16_t><<<(unsigned)blocks, 256, 0, s>>>(a);
    else
        k_w4_simple<bf16_t><<<(unsigned)blocks, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace qcnn
