// Attention over shared prefixes and 8-bit pages: the kernels of bf16 queries over i8 pages.
#include "prefix_attn.h"

namespace hydra {
namespace prefix {

template int launch_pages<bf16, i8>(const PrefixArgs&, const Shape&, hipStream_t);

}  // namespace prefix
}  // namespace hydra
