// The gradient variants of the score-modified attention for head dimensions up to 128.
#include <type_traits>

#include "score_attention_grad_tcgen05.cuh"

namespace sm120 {
SA_GRAD_INSTANTIATE(128)
}  // namespace sm120
