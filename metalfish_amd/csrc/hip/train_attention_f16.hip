// Attention with gradients in fp16.
#include "train_attention.h"

namespace mfh {
namespace attend {

hipError_t AttentionF16(const TrainAttention &a, bool backward, hipStream_t stream) {
  return ByDim<DT_F16>(a, backward, stream);
}

}  // namespace attend
}  // namespace mfh
