// Paged attention: the fp16 kernels.
#include "paged_attn.h"

namespace hydra {
namespace paged {

template int launch_group<f16>(const PagedArgs&, const Split&, const Shape&, bool, hipStream_t);

}  // namespace paged
}  // namespace hydra
