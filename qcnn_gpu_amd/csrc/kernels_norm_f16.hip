// qcnn_op_norm_res on rows of half (norm_res.h).
#include "norm_res.h"

namespace qcnn {
template hipError_t norm_res_of<f16_t>(const qcnn_norm_res_t &, hipStream_t);
}
