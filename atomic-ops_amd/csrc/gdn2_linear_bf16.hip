// The products of gdn2_linear.hpp in one type.
#include "gdn2_linear.hpp"

namespace gdn2 {
template void lin_forms<LIN_BF16>(const LinArgs&, const LinPlan&, int, int, hipStream_t);
template void lin_rows<LIN_BF16>(const LinArgs&, const LinPlan&, int, bool, bool, hipStream_t);
}  // namespace gdn2
