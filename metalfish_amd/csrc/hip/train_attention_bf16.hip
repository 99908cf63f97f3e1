// Attention with gradients in bf16.
#include "train_attention.h"

namespace mfh {
namespace attend {

hipError_t AttentionBf16(const TrainAttention &a, bool backward, hipStream_t stream) {
  return ByDim<DT_BF16>(a, backward, stream);
}

}  // namespace attend
}  // namespace mfh
