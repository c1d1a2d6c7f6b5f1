// Attention over shared prefixes and 8-bit pages: the kernels of fp32 queries over e4m3 pages.
#include "prefix_attn.h"

namespace hydra {
namespace prefix {

template int launch_pages<float, e4m3>(const PrefixArgs&, const Shape&, hipStream_t);

}  // namespace prefix
}  // namespace hydra
