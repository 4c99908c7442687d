// qcnn_op_norm_res on rows of float32 (norm_res.h).
#include "norm_res.h"

namespace qcnn {
template hipError_t norm_res_of<float>(const qcnn_norm_res_t &, hipStream_t);
}
