// Paged attention: the fp32 kernels.
#include "paged_attn.h"

namespace hydra {
namespace paged {

template int launch_group<float>(const PagedArgs&, const Split&, const Shape&, bool, hipStream_t);

}  // namespace paged
}  // namespace hydra
