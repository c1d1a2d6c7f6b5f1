// C entries of the paged attention and its bf16 kernels.
#include "paged_attn.h"

namespace hydra {
namespace paged {

template int launch_group<bf16>(const PagedArgs&, const Split&, const Shape&, bool, hipStream_t);

namespace {

int check_paged(int64_t N, int64_t H, int64_t Hkv, int64_t hd, int64_t P, int64_t page_size, int dtype) {
  HYDRA_REQUIRE(N >= 0 && H >= 1 && Hkv >= 1 && hd >= 1 && P >= 1, "paged_attn: bad size");
  HYDRA_REQUIRE(H % Hkv == 0, "paged_attn: n_heads must be a multiple of n_kv_heads");
  HYDRA_REQUIRE(hd <= 256, "paged_attn: head_dim must be at most 256");
  HYDRA_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
                "paged_attn: page_size must be a power of two in [16, 4096]");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "paged_attn: unknown dtype");
  HYDRA_REQUIRE(P <= (int64_t(1) << 30) / page_size && H < (1 << 20) && N < (int64_t(1) << 31) &&
                    N * H < (int64_t(1) << 31),
                "paged_attn: too large");
  return HYDRA_OK;
}

}  // namespace
}  // namespace paged
}  // namespace hydra

using namespace hydra;
using namespace hydra::paged;

extern "C" int hydra_paged_attn_workspace(int64_t N, int64_t Hq, int64_t Hkv, int64_t hd, int64_t P, int64_t page_size,
                                          int dtype, int64_t* bytes) {
  const int rc = check_paged(N, Hq, Hkv, hd, P, page_size, dtype);
  if (rc != HYDRA_OK) return rc;
  HYDRA_REQUIRE(bytes != nullptr, "paged_attn_workspace: null pointer");
  const Shape s = shape_of(N, Hq, Hkv, hd, dtype_size(dtype));
  *bytes = workspace_bytes(split_of(s, N, P * page_size), N, hd);
  return HYDRA_OK;
}

extern "C" int hydra_paged_attn(const void* q, const void* k_pages, const void* v_pages, void* out, const int* table,
                                int64_t table_rs, const int* lengths, int64_t N, int64_t Hq, int64_t Hkv, int64_t hd,
                                int64_t P, int64_t page_size, int64_t pages, const int64_t* q_st, const int64_t* kp_st,
                                const int64_t* vp_st, const int64_t* o_st, float scale, int dtype, void* workspace,
                                int64_t workspace_size, void* stream) {
  const int rc = check_paged(N, Hq, Hkv, hd, P, page_size, dtype);
  if (rc != HYDRA_OK) return rc;
  HYDRA_REQUIRE(pages >= 1 && pages < (int64_t(1) << 31), "paged_attn: bad number of pages");
  HYDRA_REQUIRE(table_rs >= P || N <= 1, "paged_attn: table row stride < columns");
  if (N == 0) return HYDRA_OK;
  HYDRA_REQUIRE(q && k_pages && v_pages && out && table && lengths && q_st && kp_st && vp_st && o_st,
                "paged_attn: null pointer");
  HYDRA_REQUIRE(q_st[2] == 1 && kp_st[3] == 1 && vp_st[3] == 1 && o_st[2] == 1, "paged_attn: rows need unit stride");
  const int e = dtype_size(dtype);
  const Shape s = shape_of(N, Hq, Hkv, hd, e);
  const Split p = split_of(s, N, P * page_size);
  HYDRA_REQUIRE(workspace_size >= workspace_bytes(p, N, hd) && (!p.on || (workspace && aligned16(workspace))),
                "paged_attn: workspace too small");
  PagedArgs a{};
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k_pages);
  a.v = static_cast<const char*>(v_pages);
  a.out = static_cast<char*>(out);
  bool vec = hd * e % 16 == 0 && aligned16(q) && aligned16(k_pages) && aligned16(v_pages);
  for (int i = 0; i < 2; ++i) {
    a.q_st[i] = q_st[i] * e;
    a.o_st[i] = o_st[i] * e;
    vec = vec && a.q_st[i] % 16 == 0;
  }
  for (int i = 0; i < 3; ++i) {
    a.k_st[i] = kp_st[i] * e;
    a.v_st[i] = vp_st[i] * e;
    vec = vec && (a.k_st[i] | a.v_st[i]) % 16 == 0;
  }
  HYDRA_REQUIRE(kp_st[2] >= 0 && vp_st[2] >= 0 && std::max(kp_st[2], vp_st[2]) * e * page_size < (int64_t(1) << 31),
                "paged_attn: rows of a page too far apart");
  a.table = table;
  a.lengths = lengths;
  a.table_rs = table_rs;
  a.N = static_cast<int>(N);
  a.H = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.hd = static_cast<int>(hd);
  a.G = static_cast<int>(Hq / Hkv);
  a.GB = static_cast<int>(s.gb);
  a.P = static_cast<int>(P);
  a.shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  a.pages = static_cast<int>(pages);
  a.scale = scale * kLog2e;
  a.least = p.least;
  a.plan = static_cast<int*>(workspace);
  a.part = static_cast<float*>(workspace) + (p.on ? plan_ints(N) : 0);
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int { return launch_group<T>(a, p, s, vec, st); });
}
