// RMSNorm with an 8-bit checkpoint instantiated for fp16 storage (kernels in rmsnorm8_impl.hpp).
#include "rmsnorm8_impl.hpp"

namespace pt {
namespace rmsnorm8 {
template int launch<_Float16>(bool, bool, bool, const Norm8&, void*, hipStream_t);
}  // namespace rmsnorm8
}  // namespace pt
