// Attention with gradients in fp32, and its launches.
#include "train_attention.h"

namespace mfh {
namespace attend {

hipError_t AttentionF32(const TrainAttention &a, bool backward, hipStream_t stream) {
  return ByDim<DT_F32>(a, backward, stream);
}

}  // namespace attend

namespace {

bool Sound(const TrainAttention &a) {
  return a.batch >= 0 && a.heads >= 1 && a.kv_heads >= 1 && a.heads == a.kv_heads * a.group &&
         a.q_len >= 0 && a.k_len >= 0 && a.dim >= 8 && a.dim <= 128 && a.dim % 8 == 0;
}

hipError_t Launch(const TrainAttention &a, bool backward, hipStream_t stream, std::string *err) {
  if (!Sound(a)) {
    if (err)
      *err = "attention: needs heads of 8 to 128 elements, a multiple of 8, whole groups of them a key head";
    return hipErrorInvalidValue;
  }
  if (a.dtype == DT_F32)
    return attend::AttentionF32(a, backward, stream);
  return a.dtype == DT_BF16 ? attend::AttentionBf16(a, backward, stream)
                            : attend::AttentionF16(a, backward, stream);
}

}  // namespace

std::uint64_t AttentionForwardWorkspace(const TrainAttention &a) {
  return attend::ForwardBytes(attend::ArgsOf(a, false));
}

std::uint64_t AttentionBackwardWorkspace(const TrainAttention &a) {
  const attend::Args rows = attend::ArgsOf(a, false), keys = attend::ArgsOf(a, true);
  const std::uint64_t r = attend::RowsBytes(rows), k = attend::KeysBytes(keys);
  return attend::RowValuesBytes(rows) +
         (attend::BothAtOnce(rows, keys) ? r + k : std::max(r, k));
}

hipError_t LaunchAttentionForward(const TrainAttention &a, hipStream_t stream, std::string *err) {
  return Launch(a, false, stream, err);
}

hipError_t LaunchAttentionBackward(const TrainAttention &a, hipStream_t stream, std::string *err) {
  return Launch(a, true, stream, err);
}

}  // namespace mfh
