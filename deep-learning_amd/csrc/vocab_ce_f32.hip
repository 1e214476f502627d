// The vocabulary cross entropy of fp32 tensors (two f16 planes).
#define DLMI_CE_IMPLEMENTATION
#include "vocab_ce.hpp"

namespace dlmi {
template int ce_forward<float>(dlmi_ctx *, CeArgs const &);
template int ce_backward<float>(dlmi_ctx *, CeArgs const &);
}  // namespace dlmi
