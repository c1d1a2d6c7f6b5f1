// C entries of the attention over shared prefixes and 8-bit pages.
#include "prefix_attn.h"

namespace hydra {
namespace prefix {
namespace {

// How a call is launched: pieces of up to `requests` requests, in each the
// groups' prefixes and what is behind them.
struct Pieces {
  Shape s;
  bool split;
  int64_t GB, requests, wgs;
  int waves;  // of a workgroup where it takes a whole item
  int64_t slot_a, slot_b, part_b, whole_b;  // floats; of the largest piece
};

int check_prefix(int64_t groups, int64_t N, int64_t H, int64_t Hkv, int64_t hd, int64_t P, int64_t page_size, int dtype,
                 int page_dtype) {
  HYDRA_REQUIRE(N >= 0 && groups >= 0 && H >= 1 && Hkv >= 1 && hd >= 1 && P >= 1, "prefix_attn: bad size");
  HYDRA_REQUIRE(H % Hkv == 0, "prefix_attn: n_heads must be a multiple of n_kv_heads");
  HYDRA_REQUIRE(groups == 0 || N % groups == 0, "prefix_attn: requests must be a multiple of groups");
  HYDRA_REQUIRE(hd <= 256, "prefix_attn: head_dim must be at most 256");
  HYDRA_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
                "prefix_attn: page_size must be a power of two in [16, 4096]");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "prefix_attn: unknown dtype");
  HYDRA_REQUIRE(page_dtype == dtype || page_dtype == HYDRA_PAGE_I8 || page_dtype == HYDRA_PAGE_E4M3,
                "prefix_attn: pages must be of the queries' dtype or of 8 bits");
  HYDRA_REQUIRE(page_dtype != dtype || groups > 0, "prefix_attn: pages of the queries' dtype need groups");
  HYDRA_REQUIRE(P <= (int64_t(1) << 30) / page_size && H < (1 << 20) && N < (int64_t(1) << 31) &&
                    N * H < (int64_t(1) << 31),
                "prefix_attn: too large");
  return HYDRA_OK;
}

// Split where one workgroup for each item would leave CUs idle and a request may be
// longer than a few rounds: than its waves take in two steps of 32 keys each, where items
// are few.  Measured in a graph, one workgroup an item against split, us, all requests of
// one length (ragged ones in brackets, up to that length):
//
//   4/1 heads of 64, 1 request:     1024 keys 10.3 : 9.5      2048 keys 15.0 : 9.5
//   32/8 heads of 128, 4 requests:  512 keys 12.0 : 11.6      1024 keys 16.5 : 11.9
//   4/1 heads of 256, 24 requests:  256 keys 16.6 : 17.6      512 keys 22.3 : 18.1
//   28/4 heads of 16, 24 requests:  1500 keys 10.8 : 13.0 (10.5 : 10.0)
//   32/8 heads of 128, 24 requests: 1024 keys 18.8 : 23.7 (16.2 : 16.0)
//   28/4 heads of 16, 256 requests: 2048 keys 37.6 : 42.2     4096 keys 65.8 : 71.5
//
// With many items the split costs up to a quarter where all are equally long, and only
// lengths that differ (which the host does not know) repay it.  By sizes alone, so that the
// workspace does not depend on how rows are aligned.
int pieces_of(int64_t groups, int64_t N, int64_t H, int64_t Hkv, int64_t hd, int64_t P, int64_t page_size, int dtype,
              bool vec, Pieces& p) {
  const int64_t G = H / Hkv, W = groups > 0 ? N / groups : 1, cap = P * page_size;
  p = Pieces{};
  p.s = shape_of(hd, G, W, groups > 0, dtype_size(dtype), vec);
  p.GB = (G + 15) / 16;
  const int64_t rounds = (cap + kRound - 1) / kRound;
  // rounds and rows of a launch are counted, and its threads launched, in 32 bits
  p.requests = std::min<int64_t>(std::min<int64_t>(kRequests, (int64_t(1) << 25) / H), (int64_t(1) << 29) / (rounds * Hkv * (p.GB + 1)));
  const int64_t items = N * Hkv * p.GB;
  p.waves = items > device_cus() || cap <= kRound ? 4 : whole_waves(p.s.hdp);
  const int most = whole_waves(shape_of(hd, G, W, groups > 0, dtype_size(dtype), true).hdp);
  const int64_t whole = 4 * items <= device_cus() ? most / 2 : items <= device_cus() && most == 16 ? 16 : 8;
  p.split = groups > 0 || (N <= p.requests && items < 8 * device_cus() && rounds > whole);
  HYDRA_REQUIRE(p.requests >= 1 || !p.split, "prefix_attn: too large");
  p.wgs = static_cast<int64_t>(groups > 0 ? 2 : 4) * device_cus();
  const int64_t r4 = row4(static_cast<int>(hd));
  p.slot_b = cap_b(static_cast<int>(std::min<int64_t>(G, 16))) * (2 + r4);
  if (groups > 0) {
    p.slot_a = p.s.rows_a * (2 + r4);
    const int64_t w = std::min(W, p.requests), g = std::min(groups, std::max<int64_t>(1, p.requests / W));
    p.part_b = (p.wgs + g * Hkv * ((w * G + p.s.rows_a - 1) / p.s.rows_a)) * p.slot_a;
  }
  p.whole_b = p.part_b + p.wgs * 2 * p.slot_b;
  return HYDRA_OK;
}

int64_t plan_ints() { return kPlan + 2 * kRequests + 2 + 3; }  // whole 16 bytes

int64_t workspace_bytes(const Pieces& p, int64_t groups, int64_t N, int64_t Hkv) {
  if (!p.split) return 0;
  const int64_t floats = p.whole_b + (groups > 0 ? std::min(N, p.requests) * Hkv * p.GB * p.slot_b : 0);
  return 4 * (plan_ints() / 4 * 4 + floats);
}

}  // namespace
}  // namespace prefix
}  // namespace hydra

using namespace hydra;
using namespace hydra::prefix;

extern "C" int hydra_prefix_attn_workspace(int64_t groups, int64_t N, int64_t Hq, int64_t Hkv, int64_t hd, int64_t P,
                                           int64_t page_size, int dtype, int page_dtype, int64_t* bytes) {
  int rc = check_prefix(groups, N, Hq, Hkv, hd, P, page_size, dtype, page_dtype);
  if (rc != HYDRA_OK) return rc;
  HYDRA_REQUIRE(bytes != nullptr, "prefix_attn_workspace: null pointer");
  *bytes = 0;
  if (N == 0) return HYDRA_OK;
  for (const bool vec : {true, false}) {
    Pieces p;
    rc = pieces_of(groups, N, Hq, Hkv, hd, P, page_size, dtype, vec, p);
    if (rc != HYDRA_OK) return rc;
    *bytes = std::max(*bytes, workspace_bytes(p, groups, N, Hkv));
  }
  return HYDRA_OK;
}

extern "C" int hydra_prefix_attn(const void* q, const void* k_pages, const void* v_pages, const float* k_scales,
                                 const float* v_scales, void* out, const int* table, int64_t table_rs,
                                 const int* lengths, const int* shared, int64_t groups, int64_t N, int64_t Hq,
                                 int64_t Hkv, int64_t hd, int64_t P, int64_t page_size, int64_t pages,
                                 const int64_t* q_st, const int64_t* kp_st, const int64_t* vp_st, const int64_t* ks_st,
                                 const int64_t* vs_st, const int64_t* o_st, float scale, int dtype, int page_dtype,
                                 void* workspace, int64_t workspace_size, void* stream) {
  int rc = check_prefix(groups, N, Hq, Hkv, hd, P, page_size, dtype, page_dtype);
  if (rc != HYDRA_OK) return rc;
  const bool eight = page_dtype != dtype;
  HYDRA_REQUIRE(pages >= 1 && pages < (int64_t(1) << 31), "prefix_attn: bad number of pages");
  HYDRA_REQUIRE(table_rs >= P || N <= 1, "prefix_attn: table row stride < columns");
  if (N == 0) return HYDRA_OK;
  HYDRA_REQUIRE(q && k_pages && v_pages && out && table && lengths && q_st && kp_st && vp_st && o_st &&
                    (shared || groups == 0) && (!eight || (k_scales && v_scales && ks_st && vs_st)),
                "prefix_attn: null pointer");
  HYDRA_REQUIRE(q_st[2] == 1 && kp_st[3] == 1 && vp_st[3] == 1 && o_st[2] == 1 &&
                    (!eight || (ks_st[2] == 1 && vs_st[2] == 1)),
                "prefix_attn: rows need unit stride");
  const int e = dtype_size(dtype), ep = eight ? 1 : e;
  PrefixArgs a{};
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k_pages);
  a.v = static_cast<const char*>(v_pages);
  a.out = static_cast<char*>(out);
  bool vec = hd * ep % 16 == 0 && aligned16(q) && aligned16(k_pages) && aligned16(v_pages);
  for (int i = 0; i < 2; ++i) {
    a.q_st[i] = q_st[i] * e;
    a.o_st[i] = o_st[i] * e;
    vec = vec && a.q_st[i] % 16 == 0;
    if (eight) {
      a.ks_st[i] = ks_st[i];
      a.vs_st[i] = vs_st[i];
      vec = vec && (ks_st[i] | vs_st[i]) % 4 == 0;
    }
  }
  for (int i = 0; i < 3; ++i) {
    a.k_st[i] = kp_st[i] * ep;
    a.v_st[i] = vp_st[i] * ep;
    vec = vec && (a.k_st[i] | a.v_st[i]) % 16 == 0;
  }
  HYDRA_REQUIRE(kp_st[2] >= 0 && vp_st[2] >= 0 && std::max(kp_st[2], vp_st[2]) < (int64_t(1) << 31) &&
                    std::max(kp_st[2], vp_st[2]) * ep * page_size < (int64_t(1) << 31),
                "prefix_attn: rows of a page too far apart");
  if (eight) {
    vec = vec && aligned16(k_scales) && aligned16(v_scales);
    a.ks = k_scales;
    a.vs = v_scales;
  }
  Pieces p;
  rc = pieces_of(groups, N, Hq, Hkv, hd, P, page_size, dtype, vec, p);
  if (rc != HYDRA_OK) return rc;
  HYDRA_REQUIRE(workspace_size >= workspace_bytes(p, groups, N, Hkv) &&
                    (!p.split || (workspace && aligned16(workspace))),
                "prefix_attn: workspace too small");
  a.table_rs = table_rs;
  a.H = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.hd = static_cast<int>(hd);
  a.G = static_cast<int>(Hq / Hkv);
  a.GB = static_cast<int>(p.GB);
  a.P = static_cast<int>(P);
  a.shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  a.pages = static_cast<int>(pages);
  a.scale = scale * kLog2e;
  a.split = p.split;
  a.waves = p.waves;
  a.wgs = static_cast<int>(p.wgs);
  a.cus = device_cus();
  a.plan = static_cast<int*>(workspace);
  a.part = static_cast<float*>(workspace) + plan_ints() / 4 * 4;
  a.slot_a = p.slot_a;
  a.slot_b = p.slot_b;
  a.part_b = p.part_b;
  a.whole_b = p.whole_b;
  auto st = static_cast<hipStream_t>(stream);
  auto launch = [&](const PrefixArgs& x) -> int {
    return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      if (page_dtype == HYDRA_PAGE_I8) return launch_pages<T, i8>(x, p.s, st);
      if (page_dtype == HYDRA_PAGE_E4M3) return launch_pages<T, e4m3>(x, p.s, st);
      return launch_pages<T, T>(x, p.s, st);
    });
  };
  // requests [n0, n0 + n), groups of W from group g0 on
  auto piece = [&](int64_t n0, int64_t n, int64_t g0, int64_t W) -> int {
    PrefixArgs x = a;
    x.q += n0 * a.q_st[0];
    x.out += n0 * a.o_st[0];
    x.table = table + n0 * table_rs;
    x.lengths = lengths + n0;
    x.N = static_cast<int>(n);
    x.W = static_cast<int>(W);
    x.groups = 0;
    if (groups > 0) {
      x.shared = shared + g0;
      x.groups = static_cast<int>(n / W);
      x.RB = static_cast<int>((W * a.G + p.s.rows_a - 1) / p.s.rows_a);
    }
    return launch(x);
  };
  if (groups == 0) return piece(0, N, 0, 1);
  const int64_t W = N / groups;
  if (W <= p.requests) {
    const int64_t most = p.requests / W;
    for (int64_t g = 0; g < groups; g += most) {
      const int64_t n = std::min(most, groups - g);
      rc = piece(g * W, n * W, g, W);
      if (rc != HYDRA_OK) return rc;
    }
    return HYDRA_OK;
  }
  for (int64_t g = 0; g < groups; ++g) {  // a group in pieces, each a group of its own
    for (int64_t w = 0; w < W; w += p.requests) {
      const int64_t n = std::min(p.requests, W - w);
      rc = piece(g * W + w, n, g, n);
      if (rc != HYDRA_OK) return rc;
    }
  }
  return HYDRA_OK;
}
