// ggd_battn_f32.hip -- ggd_battn.h's kernels on f32 rows (v_mfma_f32_32x32x2_f32: exact f32 products)
#include "ggd_battn_kernels.h"

namespace ggd {
namespace battn {
const Launch& battn_f32(const BtArgs& a) { return pick<float>(a); }
}  // namespace battn
}  // namespace ggd
