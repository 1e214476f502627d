// The vocabulary cross entropy of bf16 tensors (one f16 plane).
#define DLMI_CE_IMPLEMENTATION
#include "vocab_ce.hpp"

namespace dlmi {
template int ce_forward<__bf16>(dlmi_ctx *, CeArgs const &);
template int ce_backward<__bf16>(dlmi_ctx *, CeArgs const &);
}  // namespace dlmi
