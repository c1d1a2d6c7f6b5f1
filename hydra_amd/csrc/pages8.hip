// Key and value rows in pages of 8 bits on gfx950: stored with a scale for each
// row, and read back.
//
//   int8: s = max(amax / 127, 2^-126) in fp32, q = x / s rounded to nearest even;
//   e4m3: s = the least power of two >= 2^-126 with amax / s <= 448, q = x / s
//         rounded to nearest even;   x' = q s.
//
// A power of two costs e4m3 nothing (its own steps go by powers of two) and
// makes x / s exact.  int8 needs the exact quotient's rounding: amax / 2 lies in
// the middle of two values (63.5), where the quotient of two rounded numbers falls
// to either side.  So the rounding is corrected by the remainder x - q s, which
// one multiply-add gives exactly (both are multiples of the smaller unit in the
// last place and the difference is at most s).
//
// A row with an infinity or NaN gets the scale NaN and zeros: it reads back as NaN.
//
// Bound by memory: 16 bytes a lane, the lanes of a row side by side, a key and a value row
// to each group of lanes, which makes two loads in flight; more rows to a group were
// slower at every size (four: 14.9 us for both ways of 1003 rows of 4 heads of 16 in a
// graph, 102 for those below; two: 9.4 and 91; one: 6.4 and 82).  16 prompts of 4096
// rows of 8 heads of 128, bf16 and int8 (407 MB each way): 82 us for both, 9.9 TB/s, part of it
// from the last-level cache; 2 heads of 64 to e4m3 and back: 6.7 and 9.1 us.
#include "common.h"

namespace hydra {
namespace {

struct i8 { int8_t bits; };
struct e4m3 { uint8_t bits; };

constexpr float kLeastScale = 0x1p-126f;

struct Rows8Args {
  const char *k, *v;                     // rows (of a read: where they go)
  char *kp, *vp;
  float *ks, *vs;
  const int64_t *slots, *rows;           // rows: n -> row of slots (null: n)
  int64_t k_st[3], v_st[3];              // bytes: n, h, s
  int64_t kp_st[2], vp_st[2];            // bytes: page, h
  int64_t ks_st[2], vs_st[2];            // elements: page, h
  uint32_t kp_row, vp_row;
  int64_t limit;                         // slots of the pool
  int N, R, S, hd, shift;
  int lanes, log;                        // lanes of a row, their logarithm
};

// Bits of the largest |x| of E values; an infinity or NaN is at least 0x7f800000.
template <int E>
__device__ __forceinline__ uint32_t top_bits(const float* x) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) t = max(t, __float_as_uint(x[i]) & 0x7fffffffu);
  return t;
}

// The scale of a row, and its reciprocal (of int8: nearly).
template <typename KV>
__device__ __forceinline__ void scale_of(uint32_t top, float& s, float& inv) {
  if (top >= 0x7f800000u) {
    s = __uint_as_float(0x7fc00000u);
    inv = 0.f;
  } else if constexpr (std::is_same<KV, i8>::value) {
    s = fmaxf(__uint_as_float(top) / 127.f, kLeastScale);
    inv = 1.f / s;
  } else {
    const int e = static_cast<int>(top >> 23) - ((top & 0x7fffffu) > 0x600000u ? 7 : 8);  // 448 = 1.75 x 2^8
    const uint32_t b = static_cast<uint32_t>(max(e, 1));
    s = __uint_as_float(b << 23);
    inv = __uint_as_float((254u - b) << 23);
  }
}

__device__ __forceinline__ int to_i8(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r2 = 2.f * fmaf(-q, s, x);  // twice the remainder, exactly
  const bool odd = static_cast<int>(q) & 1;
  if (r2 > s || (r2 == s && odd)) q += 1.f;
  if (r2 < -s || (r2 == -s && odd)) q -= 1.f;
  return static_cast<int>(fminf(fmaxf(q, -127.f), 127.f));
}

// E values as E bytes, in words; a row that is not finite (its scale NaN) as zeros.
template <typename KV, int E>
__device__ __forceinline__ void to_bytes(const float* x, float s, float inv, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    if constexpr (std::is_same<KV, i8>::value) {
      uint32_t b = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) b |= (static_cast<uint32_t>(to_i8(x[4 * i + j], s, inv)) & 0xffu) << (8 * j);
      w[i] = b;
    } else {
      int b = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
      w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, b, true));
    }
    if (s != s) w[i] = 0;
  }
}

// Elements [piece E, +E) of a row; zeros past its end.
template <typename T, bool VEC>
__device__ __forceinline__ void row_values(const char* row, int piece, int hd, float* x) {
  constexpr int E = Vec<T>::N;
  if constexpr (VEC) {
    if (piece * E < hd) {
      load16<T>(reinterpret_cast<const T*>(row) + piece * E, x);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    x[i] = !VEC && piece * E + i < hd ? to_f32(reinterpret_cast<const T*>(row)[piece * E + i]) : 0.f;
}

template <int E, bool VEC>
__device__ __forceinline__ void put_bytes(char* row, int piece, int hd, const uint32_t* w) {
  if constexpr (VEC) {
    if (piece * E < hd) {
      if constexpr (E == 8) *reinterpret_cast<uint2*>(row + piece * E) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(row + piece * E) = w[0];
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (piece * E + i < hd) row[piece * E + i] = static_cast<char>(w[i / 4] >> (8 * (i % 4)));
  }
}

template <typename T, typename KV, bool VEC>
__global__ __launch_bounds__(256) void store8_kernel(Rows8Args a) {
  constexpr int E = Vec<T>::N;
  const int piece = threadIdx.x & (a.lanes - 1), group = threadIdx.x >> a.log, groups = 256 >> a.log;
  const int h = blockIdx.y;
  for (int n = blockIdx.z; n < a.N; n += gridDim.z) {
    const int64_t r = a.rows ? a.rows[n] : n;
    if (r < 0 || r >= a.R) continue;
    const int64_t* slots = a.slots + r * a.S;
    const char *k = a.k + n * a.k_st[0] + h * a.k_st[1], *v = a.v + n * a.v_st[0] + h * a.v_st[1];
    const int64_t s = static_cast<int64_t>(blockIdx.x) * groups + group, slot = s < a.S ? slots[s] : -1;
    if (slot < 0 || slot >= a.limit) continue;  // the lanes of a group together
    float x[2][E];
    row_values<T, VEC>(k + s * a.k_st[2], piece, a.hd, x[0]);
    row_values<T, VEC>(v + s * a.v_st[2], piece, a.hd, x[1]);
    const int64_t page = slot >> a.shift;
    const uint32_t row = static_cast<uint32_t>(slot) & ((1u << a.shift) - 1);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t top = top_bits<E>(x[c]);
      for (int off = a.lanes >> 1; off > 0; off >>= 1)
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off)));
      float scale, inv;
      uint32_t w[E / 4];
      scale_of<KV>(top, scale, inv);
      to_bytes<KV, E>(x[c], scale, inv, w);
      char* to = c ? a.vp + page * a.vp_st[0] + h * a.vp_st[1] + static_cast<uint64_t>(row) * a.vp_row
                   : a.kp + page * a.kp_st[0] + h * a.kp_st[1] + static_cast<uint64_t>(row) * a.kp_row;
      put_bytes<E, VEC>(to, piece, a.hd, w);
      if (piece == 0)
        (c ? a.vs[page * a.vs_st[0] + h * a.vs_st[1] + row] : a.ks[page * a.ks_st[0] + h * a.ks_st[1] + row]) = scale;
    }
  }
}

// Four values of a word of 8 bits.
template <typename KV>
__device__ __forceinline__ void from_word(uint32_t w, float s, float* x) {
  if constexpr (std::is_same<KV, i8>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * s;
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = lo[0] * s, x[1] = lo[1] * s, x[2] = hi[0] * s, x[3] = hi[1] * s;
  }
}

// Rows out of their pages, into k and v.  A lane writes 16 bytes of a row (an
// element where rows are not made of such).
template <typename T, typename KV, bool VEC>
__global__ __launch_bounds__(256) void read_kernel(Rows8Args a) {
  constexpr int E = VEC ? Vec<T>::N : 1;
  constexpr bool EIGHT = sizeof(KV) == 1;
  const int lane = threadIdx.x & (a.lanes - 1), group = threadIdx.x >> a.log, groups = 256 >> a.log;
  const int h = blockIdx.y;
  const int64_t s = static_cast<int64_t>(blockIdx.x) * groups + group;
  if (s >= a.S) return;
  for (int n = blockIdx.z; n < a.N; n += gridDim.z) {
    const int64_t r = a.rows ? a.rows[n] : n;
    const int64_t slot = r >= 0 && r < a.R ? a.slots[r * a.S + s] : -1;
    const bool in = slot >= 0 && slot < a.limit;
    const int64_t page = in ? slot >> a.shift : 0;
    const uint32_t row = in ? static_cast<uint32_t>(slot) & ((1u << a.shift) - 1) : 0;
    float scale[2] = {1.f, 1.f};
    if constexpr (EIGHT) {
      scale[0] = a.ks[page * a.ks_st[0] + h * a.ks_st[1] + row];
      scale[1] = a.vs[page * a.vs_st[0] + h * a.vs_st[1] + row];
    }
    for (int piece = lane; piece * E < a.hd; piece += a.lanes) {
      float x[2][E];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const char* p = (c ? a.vp + page * a.vp_st[0] + h * a.vp_st[1] + static_cast<uint64_t>(row) * a.vp_row
                           : a.kp + page * a.kp_st[0] + h * a.kp_st[1] + static_cast<uint64_t>(row) * a.kp_row) +
                        static_cast<int64_t>(piece) * E * static_cast<int>(sizeof(KV));
        if constexpr (!VEC) {
          if constexpr (EIGHT) {
            float f[4];
            from_word<KV>(*reinterpret_cast<const uint8_t*>(p), scale[c], f);
            x[c][0] = f[0];
          } else {
            x[c][0] = to_f32(*reinterpret_cast<const T*>(p));
          }
        } else if constexpr (EIGHT) {
#pragma unroll
          for (int i = 0; i < E / 4; ++i) from_word<KV>(reinterpret_cast<const uint32_t*>(p)[i], scale[c], x[c] + 4 * i);
        } else {
          load16<T>(reinterpret_cast<const T*>(p), x[c]);
        }
        if (!in) {
#pragma unroll
          for (int i = 0; i < E; ++i) x[c][i] = 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        T* to = reinterpret_cast<T*>(const_cast<char*>(c ? a.v + n * a.v_st[0] + h * a.v_st[1] + s * a.v_st[2]
                                                         : a.k + n * a.k_st[0] + h * a.k_st[1] + s * a.k_st[2])) +
                static_cast<int64_t>(piece) * E;
        if constexpr (VEC) store16<T, true>(to, x[c]);
        else *to = from_f32<T>(x[c][0]);
      }
    }
  }
}

int page_shift(int64_t page_size) {
  for (int s = 4; s <= 12; ++s)
    if (page_size == (int64_t(1) << s)) return s;
  return -1;
}

// What both entries check and lay out; `vec` gets whether 16-byte pieces of rows of
// dtype and the bytes beside them are aligned.
int fill_args(Rows8Args& a, bool& vec, const char* name, const void* k, const void* v, const void* k_pages,
              const void* v_pages, const float* k_scales, const float* v_scales, const int64_t* slots, int64_t R,
              const int64_t* rows, int64_t N, int64_t Hkv, int64_t S, int64_t hd, int64_t pages, int64_t page_size,
              const int64_t* k_st, const int64_t* v_st, const int64_t* kp_st, const int64_t* vp_st,
              const int64_t* ks_st, const int64_t* vs_st, int dtype, int page_dtype) {
  const std::string at(name);
  HYDRA_REQUIRE(N >= 0 && S >= 0 && R >= 0 && Hkv >= 1 && hd >= 1 && pages >= 1, at + ": bad size");
  HYDRA_REQUIRE(rows || R >= N, at + ": fewer rows of slots than prompts");
  const int shift = page_shift(page_size);
  HYDRA_REQUIRE(shift >= 0, at + ": page_size must be a power of two in [16, 4096]");
  const int e = dtype_size(dtype);
  HYDRA_REQUIRE(e > 0, at + ": unknown dtype");
  const bool eight = page_dtype == HYDRA_PAGE_I8 || page_dtype == HYDRA_PAGE_E4M3;
  HYDRA_REQUIRE(eight || page_dtype == dtype, at + ": pages must be of the rows' dtype or of 8 bits");
  HYDRA_REQUIRE(N < (int64_t(1) << 31) && R < (int64_t(1) << 31) && S < (int64_t(1) << 31) && Hkv <= 65535 &&
                    hd <= 256 && pages < (int64_t(1) << 31),
                at + ": too large");
  if (N == 0 || S == 0) return HYDRA_OK;
  HYDRA_REQUIRE(k && v && k_pages && v_pages && slots && k_st && v_st && kp_st && vp_st &&
                    (!eight || (k_scales && v_scales && ks_st && vs_st)),
                at + ": null pointer");
  HYDRA_REQUIRE(k_st[3] == 1 && v_st[3] == 1 && kp_st[3] == 1 && vp_st[3] == 1 &&
                    (!eight || (ks_st[2] == 1 && vs_st[2] == 1)),
                at + ": rows need unit stride");
  const int ep = eight ? 1 : e, piece = 16 / e * ep;  // bytes of a piece in a page
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.kp = static_cast<char*>(const_cast<void*>(k_pages));
  a.vp = static_cast<char*>(const_cast<void*>(v_pages));
  a.ks = const_cast<float*>(k_scales);
  a.vs = const_cast<float*>(v_scales);
  a.slots = slots;
  a.rows = rows;
  a.limit = pages * page_size;
  a.N = static_cast<int>(N);
  a.R = static_cast<int>(R);
  a.S = static_cast<int>(S);
  a.hd = static_cast<int>(hd);
  a.shift = shift;
  vec = hd * e % 16 == 0 && aligned16(k) && aligned16(v) && aligned16(k_pages) && aligned16(v_pages);
  for (int i = 0; i < 3; ++i) {
    a.k_st[i] = k_st[i] * e;
    a.v_st[i] = v_st[i] * e;
    vec = vec && (a.k_st[i] | a.v_st[i]) % 16 == 0;
  }
  for (int i = 0; i < 2; ++i) {
    a.kp_st[i] = kp_st[i] * ep;
    a.vp_st[i] = vp_st[i] * ep;
    vec = vec && (a.kp_st[i] | a.vp_st[i]) % piece == 0;
    if (eight) {
      a.ks_st[i] = ks_st[i];
      a.vs_st[i] = vs_st[i];
    }
  }
  HYDRA_REQUIRE(kp_st[2] >= 0 && vp_st[2] >= 0 && kp_st[2] < (int64_t(1) << 32) / ep && vp_st[2] < (int64_t(1) << 32) / ep,
                at + ": rows too far apart");
  a.kp_row = static_cast<uint32_t>(kp_st[2] * ep);
  a.vp_row = static_cast<uint32_t>(vp_st[2] * ep);
  vec = vec && (a.kp_row | a.vp_row) % piece == 0;
  return HYDRA_OK;
}

// Lanes of a row of `pieces`: a power of two, at most a wave.
void set_lanes(Rows8Args& a, int64_t pieces) {
  a.log = 0;
  while ((1 << a.log) < pieces && a.log < 6) ++a.log;
  a.lanes = 1 << a.log;
}

dim3 grid_of(const Rows8Args& a, int64_t Hkv) {
  const int64_t span = 256 >> a.log;
  return dim3(static_cast<unsigned>((a.S + span - 1) / span), static_cast<unsigned>(Hkv),
              static_cast<unsigned>(a.N < 65535 ? a.N : 65535));
}

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int hydra_page_store8(const void* k, const void* v, void* k_pages, void* v_pages, float* k_scales,
                                 float* v_scales, const int64_t* slots, int64_t R, const int64_t* rows, int64_t N,
                                 int64_t Hkv, int64_t S, int64_t hd, int64_t pages, int64_t page_size,
                                 const int64_t* k_st, const int64_t* v_st, const int64_t* kp_st, const int64_t* vp_st,
                                 const int64_t* ks_st, const int64_t* vs_st, int dtype, int page_dtype, void* stream) {
  Rows8Args a{};
  bool vec = false;
  HYDRA_REQUIRE(page_dtype == HYDRA_PAGE_I8 || page_dtype == HYDRA_PAGE_E4M3, "page_store8: pages must be of 8 bits");
  const int rc = fill_args(a, vec, "page_store8", k, v, k_pages, v_pages, k_scales, v_scales, slots, R, rows, N, Hkv, S,
                           hd, pages, page_size, k_st, v_st, kp_st, vp_st, ks_st, vs_st, dtype, page_dtype);
  if (rc != HYDRA_OK || N == 0 || S == 0) return rc;
  const int e = dtype_size(dtype);
  set_lanes(a, (hd * e + 15) / 16);
  const dim3 grid = grid_of(a, Hkv);
  HYDRA_REQUIRE(grid_fits(grid.x, 256), "page_store8: too large");
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    if (page_dtype == HYDRA_PAGE_I8) {
      if (vec) store8_kernel<T, i8, true><<<grid, 256, 0, st>>>(a);
      else store8_kernel<T, i8, false><<<grid, 256, 0, st>>>(a);
    } else {
      if (vec) store8_kernel<T, e4m3, true><<<grid, 256, 0, st>>>(a);
      else store8_kernel<T, e4m3, false><<<grid, 256, 0, st>>>(a);
    }
    return check_launch("page_store8");
  });
}

extern "C" int hydra_page_read(const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                               void* k, void* v, const int64_t* slots, int64_t R, const int64_t* rows, int64_t N,
                               int64_t Hkv, int64_t S, int64_t hd, int64_t pages, int64_t page_size,
                               const int64_t* kp_st, const int64_t* vp_st, const int64_t* ks_st, const int64_t* vs_st,
                               const int64_t* k_st, const int64_t* v_st, int dtype, int page_dtype, void* stream) {
  Rows8Args a{};
  bool vec = false;
  const int rc = fill_args(a, vec, "page_read", k, v, k_pages, v_pages, k_scales, v_scales, slots, R, rows, N, Hkv, S,
                           hd, pages, page_size, k_st, v_st, kp_st, vp_st, ks_st, vs_st, dtype, page_dtype);
  if (rc != HYDRA_OK || N == 0 || S == 0) return rc;
  const int e = dtype_size(dtype);
  set_lanes(a, vec ? hd * e / 16 : hd);
  const dim3 grid = grid_of(a, Hkv);
  HYDRA_REQUIRE(grid_fits(grid.x, 256), "page_read: too large");
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    if (page_dtype == HYDRA_PAGE_I8) {
      if (vec) read_kernel<T, i8, true><<<grid, 256, 0, st>>>(a);
      else read_kernel<T, i8, false><<<grid, 256, 0, st>>>(a);
    } else if (page_dtype == HYDRA_PAGE_E4M3) {
      if (vec) read_kernel<T, e4m3, true><<<grid, 256, 0, st>>>(a);
      else read_kernel<T, e4m3, false><<<grid, 256, 0, st>>>(a);
    } else {
      if (vec) read_kernel<T, T, true><<<grid, 256, 0, st>>>(a);
      else read_kernel<T, T, false><<<grid, 256, 0, st>>>(a);
    }
    return check_launch("page_read");
  });
}
