// Attention over shared prefixes and 8-bit pages: the kernels of fp16 queries over fp16 pages.
#include "prefix_attn.h"

namespace hydra {
namespace prefix {

template int launch_pages<f16, f16>(const PrefixArgs&, const Shape&, hipStream_t);

}  // namespace prefix
}  // namespace hydra
