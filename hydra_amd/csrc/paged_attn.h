// Attention of one new token per request over a paged key-value cache, gfx950.
//
//   o[n,h] = sum_t p_t v[t, h/G],  p = softmax_t(scale q[n,h] . k[t, h/G]),
//   t < lengths[n], position t in page table[n, t / page_size].
//
// A step reads each key and value once and does 4 G flops per element pair:
// HBM-bound at every group size up to 16.  A wave walks its keys KT at a time:
//
//  * scores S^T = K Q^T on the matrix cores: keys are the rows of the A operand,
//    loaded from the pages in the operand's own layout (16 bytes a lane), the up
//    to GP heads of the group are columns of B (the others zero).  The order of
//    the head dimension inside an operand is free as long as K and Q agree, so
//    each lane's 16 bytes are one operand of a 16-bit type (16x16x32) and four
//    of fp32 (16x16x4, full fp32 products);
//  * the softmax keeps each head's running maximum (fp32, log2 units) in the
//    lanes of its column; the sums of one lane's keys are added up at the end;
//  * P goes through 4 KT GP bytes of LDS to the lanes that hold the rows of V,
//    which accumulate p v in fp32 with plain multiply-adds: P is never rounded,
//    V needs no transposed copy, and G multiply-adds per value stay below the
//    time its bytes take (G = 8: about a third).
//
// Pages hold 16 rows or more, so the 16 keys of an operand lie in one page and
// page ids are wave-uniform scalar loads.  An entry outside the pool counts as
// absent: its keys are not seen.  Rows past a request's length are loaded at
// most within their own page and stay out of both sums, whatever they hold.
//
// Split: the keys of all (request, key head, head block) items are laid end to
// end in rounds of 4 KT keys (one tile per wave) and dealt out evenly to the
// workgroups, whatever the lengths; an item that more than one of them works on
// leaves (max, sum, unscaled output) per part in the workspace, and a second
// kernel joins them in order.  No atomics: the same inputs give the same bits.
#pragma once
#include "common.h"
#include "mod_keys.h"

#include <algorithm>

namespace hydra {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxRequests = 2048;  // of the split form: prefix sums of their rounds lie in LDS
constexpr int kMaxParts = 256;      // of one item

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

struct PagedArgs {
  const char *q, *k, *v;
  char* out;
  int64_t q_st[2], o_st[2];         // bytes: n, h
  int64_t k_st[3], v_st[3];         // bytes: page, h, row
  const int* table;
  const int* lengths;
  int64_t table_rs;
  int N, H, Hkv, hd, G, GB, P, shift, pages;
  float scale;                       // times log2(e)
  // split form: rounds of a workgroup at least, workgroups, results
  int least, groups;
  int* plan;                         // [0] rounds per workgroup, [1 + n] prefix of rounds
  float* part;                       // [groups][2][GP (2 + hd)]
};

template <typename T>
__device__ __forceinline__ f32x4_t mfma16(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  } else if constexpr (std::is_same<T, f16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}

// Piece `piece` (16 bytes) of a row of hd elements; zeros past its end.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 row_piece(const char* row, int piece, int hd) {
  constexpr int E = Vec<T>::N;
  if constexpr (VEC) {
    return piece * E < hd ? *reinterpret_cast<const uint4*>(row + piece * 16) : make_uint4(0, 0, 0, 0);
  } else {
    const T* p = reinterpret_cast<const T*>(row) + piece * E;
    float f[E];
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = piece * E + i < hd ? to_f32(p[i]) : 0.f;
    return pack16<T>(f);  // exact: the values are T's
  }
}

// Keys of request n: its length, within what its table row can hold.
__device__ __forceinline__ int seen_keys(const PagedArgs& a, int n) {
  return max(0, min(a.lengths[n], a.P << a.shift));
}

// Keys of a wave's step: 4 to 8 KB of keys and as much of values in flight.
constexpr int tile_keys(int lpr) { return lpr <= 4 ? 64 : (lpr <= 16 ? 32 : 16); }
template <int LPR> struct Tile { static constexpr int KT = tile_keys(LPR); };

// One item's keys [t0, t1) rounds -> per-head max, sum and output of the whole
// workgroup in LDS (acc[GP][hdp], then m[GP], l[GP]).
template <typename T, int GP, int LPR, bool VEC>
__device__ __forceinline__ void item_keys(const PagedArgs& a, int n, int h, int gb, int t0, int t1, float* sm) {
  constexpr int KT = Tile<LPR>::KT, E = Vec<T>::N, NC = LPR < 4 ? 1 : LPR / 4;
  constexpr int RPI = 64 / LPR;          // rows that one V load of the wave covers
  constexpr int NV = KT / RPI, NB = KT / 16;
  constexpr int HDP = LPR * E;           // hd rounded up
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4;  // operand row / column, 16-byte piece
  const int heads = min(GP, a.G - gb * GP);
  const int len = seen_keys(a, n);
  float* plds = sm + wave * KT * GP;

  uint4 qf[NC];
  {
    const char* qrow = a.q + n * a.q_st[0] + static_cast<int64_t>(h * a.G + gb * GP + (col < heads ? col : 0)) * a.q_st[1];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qf[c] = row_piece<T, VEC>(qrow, 4 * c + g4, a.hd);
      if (col >= heads) qf[c] = make_uint4(0, 0, 0, 0);
    }
  }
  float m = -INFINITY, l = 0.f;
  float acc[GP][E];
#pragma unroll
  for (int g = 0; g < GP; ++g)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[g][e] = 0.f;

  const int* trow = a.table + n * a.table_rs;
  const int vrow = lane / LPR, vpiece = lane % LPR;
  for (int t = t0; t < t1; ++t) {
    const int key0 = (t * 4 + wave) * KT;
    if (key0 >= len) break;
    // page of each 16 keys, wave-uniform; -1: not there
    int page[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int key = __builtin_amdgcn_readfirstlane(key0 + 16 * b);
      int p = key < len ? trow[key >> a.shift] : -1;
      page[b] = static_cast<unsigned>(p) < static_cast<unsigned>(a.pages) ? p : -1;
    }
    const int rmask = (1 << a.shift) - 1;
    uint4 kf[NB][NC];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const char* base = a.k + max(page[b], 0) * a.k_st[0] + h * a.k_st[1] +
                         static_cast<int64_t>(((key0 + 16 * b) & rmask) + col) * a.k_st[2];
#pragma unroll
      for (int c = 0; c < NC; ++c) kf[b][c] = row_piece<T, VEC>(base, 4 * c + g4, a.hd);
    }
    uint4 vf[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int row = i * RPI + vrow;
      int p = page[i * RPI / 16];
      if constexpr (RPI == 32) p = vrow < 16 ? p : page[i * RPI / 16 + 1];
      const int key = key0 + row;
      const bool seen = key < len && p >= 0;
      const char* base = a.v + max(p, 0) * a.v_st[0] + h * a.v_st[1] + static_cast<int64_t>(key & rmask) * a.v_st[2];
      vf[i] = row_piece<T, VEC>(base, vpiece, a.hd);
      if (!seen) vf[i] = make_uint4(0, 0, 0, 0);  // 0 x whatever lies there must add nothing
    }
    f32x4_t s[NB];
    float top = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      s[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) s[b] = mfma16<T>(kf[b][c], qf[c], s[b]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = key0 + 16 * b + 4 * g4 + r;
        s[b][r] = key < len && page[b] >= 0 ? s[b][r] * a.scale : -INFINITY;
        top = fmaxf(top, s[b][r]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    if (__any(top > m)) {
      const float mn = fmaxf(m, top);
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float al = __shfl(alpha, g);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[g][e] *= al;
      }
    }
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f(s[b][r] - ms);
        l += p;
        if (col < GP) plds[(16 * b + 4 * g4 + r) * GP + col] = p;
      }
    // P is read by other lanes of this wave alone; its LDS operations keep their order.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float p[GP], v[E];
#pragma unroll
      for (int g = 0; g < GP; ++g) p[g] = plds[(i * RPI + vrow) * GP + g];
      unpack16<T>(vf[i], v);
#pragma unroll
      for (int g = 0; g < GP; ++g)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[g][e] = fmaf(p[g], v[e], acc[g][e]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // The wave's own sums ...
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int off = LPR; off < 64; off <<= 1)
#pragma unroll
    for (int g = 0; g < GP; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] += __shfl_xor(acc[g][e], off);
  // ... then the four waves', in order.
  float* wm = sm;                 // [4][GP] max, [4][GP] sum, [4][GP][HDP] output
  float* wl = sm + 4 * GP;
  float* wa = sm + 8 * GP;
  __syncthreads();                // P's memory is free
  if (lane < GP) {
    wm[wave * GP + lane] = m;
    wl[wave * GP + lane] = l;
  }
  if (lane < LPR) {
#pragma unroll
    for (int g = 0; g < GP; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) wa[(wave * GP + g) * HDP + lane * E + e] = acc[g][e];
  }
  __syncthreads();
}

// The four waves' results of item_keys as (max, sum, output element) of head g.
template <int GP, int HDP>
__device__ __forceinline__ void join_waves(const float* sm, int g, int d, float& m, float& l, float& o) {
  m = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, sm[w * GP + g]);
  const float ms = m == -INFINITY ? 0.f : m;
  l = 0.f;
  o = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float c = __builtin_amdgcn_exp2f(sm[w * GP + g] - ms);
    l = fmaf(c, sm[4 * GP + w * GP + g], l);
    o = fmaf(c, sm[8 * GP + (w * GP + g) * HDP + d], o);
  }
}

template <int GP, int LPR, typename T>
constexpr int lds_floats() {
  constexpr int p = 4 * Tile<LPR>::KT * GP, j = 8 * GP + 4 * GP * LPR * Vec<T>::N;
  return p > j ? p : j;
}

template <typename T>
__device__ __forceinline__ T* out_row(const PagedArgs& a, int n, int head) {
  return reinterpret_cast<T*>(a.out + n * a.o_st[0] + static_cast<int64_t>(head) * a.o_st[1]);
}

template <int LPR>
__device__ __forceinline__ int rounds_of(int len) {
  constexpr int R = 4 * Tile<LPR>::KT;
  return len / R + (len % R != 0);
}

// The workgroup's whole item, normalised; a request without keys gets zeros.
template <typename T, int GP, int HDP>
__device__ __forceinline__ void write_out(const PagedArgs& a, int n, int h, int gb, const float* sm) {
  const int heads = min(GP, a.G - gb * GP);
  for (int e = threadIdx.x; e < heads * a.hd; e += 256) {
    const int g = e / a.hd, d = e - g * a.hd;
    float m, l, o;
    join_waves<GP, HDP>(sm, g, d, m, l, o);
    out_row<T>(a, n, h * a.G + gb * GP + g)[d] = from_f32<T>(l == 0.f ? 0.f : o / l);
  }
}

// One workgroup per item, no split.
template <typename T, int GP, int LPR, bool VEC>
__global__ __launch_bounds__(256) void paged_attn_whole_kernel(PagedArgs a) {
  constexpr int HDP = LPR * Vec<T>::N;
  __shared__ __attribute__((aligned(16))) float sm[lds_floats<GP, LPR, T>()];
  const int item = blockIdx.x, gb = item % a.GB, h = item / a.GB % a.Hkv, n = item / a.GB / a.Hkv;
  item_keys<T, GP, LPR, VEC>(a, n, h, gb, 0, rounds_of<LPR>(seen_keys(a, n)), sm);
  write_out<T, GP, HDP>(a, n, h, gb, sm);
}

// Split form: workgroup w works on the rounds [w per, (w+1) per) of all items.
template <typename T, int GP, int LPR, bool VEC>
__global__ __launch_bounds__(256) void paged_attn_split_kernel(PagedArgs a) {
  constexpr int HDP = LPR * Vec<T>::N;
  __shared__ __attribute__((aligned(16))) float sm[lds_floats<GP, LPR, T>()];
  __shared__ int pre[kMaxRequests + 1];
  __shared__ int wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // prefix sums of the requests' rounds
  int base = 0;
  if (tid == 0) pre[0] = 0;
  for (int i0 = 0; i0 < a.N; i0 += 256) {
    const int i = i0 + tid;
    int s = wave_incl_sum(i < a.N ? rounds_of<LPR>(seen_keys(a, i)) : 0);
    if (lane == 63) wsum[wave] = s;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) s += wsum[w];
      all += wsum[w];
    }
    if (i < a.N) pre[i + 1] = base + s;
    base += all;
    __syncthreads();
  }
  const int HG = a.Hkv * a.GB, total = base * HG;
  const int per = max(a.least, (total + a.groups - 1) / a.groups);
  if (blockIdx.x == 0) {  // for the joining kernel
    if (tid == 0) a.plan[0] = per;
    for (int i = tid; i <= a.N; i += 256) a.plan[1 + i] = pre[i];
  }
  // the last workgroup's range may pass int only if the total does (checked on the host)
  const int begin = min(static_cast<int64_t>(blockIdx.x) * per, static_cast<int64_t>(total));
  const int end = min(static_cast<int64_t>(begin) + per, static_cast<int64_t>(total));
  int n = 0;
  if (begin < end) {  // the last n with pre[n] HG <= begin
    int hi = a.N;
    while (hi - n > 1) {
      const int mid = (n + hi) >> 1;
      if (pre[mid] * HG <= begin) n = mid; else hi = mid;
    }
  }
  for (int u = begin; u < end;) {
    while (pre[n + 1] * HG <= u) ++n;
    const int r = pre[n + 1] - pre[n], at = u - pre[n] * HG, hg = at / r, t0 = at - hg * r;
    const int count = min(r - t0, end - u), h = hg / a.GB, gb = hg - h * a.GB;
    item_keys<T, GP, LPR, VEC>(a, n, h, gb, t0, t0 + count, sm);
    if (count == r) {
      write_out<T, GP, HDP>(a, n, h, gb, sm);
    } else {
      float* part = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (u == begin ? 0 : 1)) * GP * (2 + a.hd);
      for (int e = tid; e < GP * a.hd; e += 256) {
        const int g = e / a.hd, d = e - g * a.hd;
        float m, l, o;
        join_waves<GP, HDP>(sm, g, d, m, l, o);
        part[2 * GP + e] = o;
        if (d == 0) {
          part[g] = m;
          part[GP + g] = l;
        }
      }
    }
    u += count;
    __syncthreads();
  }
}

// Joins the parts of one item, in their order; writes the zeros of a request
// without keys.  Items that one workgroup had whole are written already.
template <typename T, int GP>
__global__ __launch_bounds__(1024) void paged_attn_join_kernel(PagedArgs a) {
  __shared__ float weight[GP][kMaxParts];
  __shared__ float sums[1024];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int HG = a.Hkv * a.GB, n = blockIdx.x / HG, hg = blockIdx.x - n * HG, h = hg / a.GB, gb = hg - h * a.GB;
  const int per = a.plan[0], p0 = a.plan[1 + n], r = a.plan[2 + n] - p0;
  const int heads = min(GP, a.G - gb * GP);
  const int u0 = p0 * HG + hg * r, w0 = u0 / per, parts = r == 0 ? 0 : (u0 + r - 1) / per - w0 + 1;
  if (parts == 1) return;
  const int size = GP * (2 + a.hd);
  auto part = [&](int p) {  // only the first one can begin inside its workgroup's range
    return a.part + (static_cast<int64_t>(w0 + p) * 2 + (p == 0 && u0 != w0 * per ? 1 : 0)) * size;
  };
  for (int g = wave; g < GP; g += 16) {
    float m = -INFINITY;
    for (int p = lane; p < parts; p += 64) m = fmaxf(m, part(p)[g]);
    m = wave_max(m);
    const float ms = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int p = lane; p < parts; p += 64) l += __builtin_amdgcn_exp2f(part(p)[g] - ms) * part(p)[GP + g];
    l = wave_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int p = lane; p < parts; p += 64) weight[g][p] = __builtin_amdgcn_exp2f(part(p)[g] - ms) * inv;
  }
  __syncthreads();
  // elements of the item side by side, the parts dealt out over what is left of the workgroup
  const int elems = heads * a.hd;
  int lanes = 1;  // threads of one element
  while (lanes * 2 * elems <= 1024) lanes *= 2;
  const int step = 1024 / lanes, sub = tid / step;
  for (int e0 = 0; e0 < elems; e0 += step) {
    const int e = e0 + tid - sub * step;
    float o = 0.f;
    if (e < elems) {
      const int g = e / a.hd;
#pragma unroll 8
      for (int p = sub; p < parts; p += lanes) o = fmaf(weight[g][p], part(p)[2 * GP + e], o);
    }
    sums[tid] = o;
    __syncthreads();
    if (sub == 0 && e < elems) {
      for (int i = 1; i < lanes; ++i) o += sums[i * step + tid];
      const int g = e / a.hd;
      out_row<T>(a, n, h * a.G + gb * GP + g)[e - g * a.hd] = from_f32<T>(o);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------- launch
struct Shape {
  int gp, lpr, kt;
  int64_t gb, items;
};

// Heads of a block: the smallest power of two that holds the group, at most 8
// (a larger group takes more blocks, which read its keys again, from L2).
// Lanes of a row: its 16-byte pieces, rounded up to a power of two.
inline Shape shape_of(int64_t N, int64_t H, int64_t Hkv, int64_t hd, int e) {
  Shape s{};
  const int64_t G = H / Hkv;
  s.gp = 1;
  while (s.gp < 8 && s.gp < G) s.gp *= 2;
  s.gb = (G + s.gp - 1) / s.gp;
  s.lpr = 2;
  while (s.lpr * 16 < hd * e) s.lpr *= 2;
  s.kt = tile_keys(s.lpr);
  s.items = N * Hkv * s.gb;
  return s;
}

struct Split {
  bool on;
  int least, groups;
};

// Split where the items alone would not fill the chip and a request may be
// longer than one workgroup's least share.
inline Split split_of(const Shape& s, int64_t N, int64_t capacity) {
  const int64_t round = 4 * s.kt, most = (capacity + round - 1) / round;
  Split r{};
  r.groups = 4 * device_cus();
  const int64_t least = std::max<int64_t>(2, (most + kMaxParts - 2) / (kMaxParts - 1));
  r.on = N <= kMaxRequests && s.items < 8 * device_cus() && most > least && most * s.items < (int64_t(1) << 31);
  r.least = static_cast<int>(std::min<int64_t>(least, 1 << 30));
  return r;
}

// The plan's whole numbers, rounded up to 16 bytes.
inline int64_t plan_ints(int64_t N) { return (N + 2 + 3) / 4 * 4; }

inline int64_t workspace_bytes(const Split& p, int64_t N, int64_t hd) {
  if (!p.on) return 0;
  return 4 * (plan_ints(N) + static_cast<int64_t>(p.groups) * 2 * 8 * (2 + hd));
}

// Rows that 16-byte loads cannot take come through one form, of 8 heads.
template <typename T, int GP, int LPR>
int launch_paged(const PagedArgs& a, const Split& p, int64_t items, bool vec, hipStream_t st) {
  if constexpr (GP == 8) {
    if (!vec) {
      if (p.on) paged_attn_split_kernel<T, GP, LPR, false><<<p.groups, 256, 0, st>>>(a);
      else paged_attn_whole_kernel<T, GP, LPR, false><<<static_cast<unsigned>(items), 256, 0, st>>>(a);
    }
  }
  if (p.on) {
    if (vec) paged_attn_split_kernel<T, GP, LPR, true><<<p.groups, 256, 0, st>>>(a);
    paged_attn_join_kernel<T, GP><<<static_cast<unsigned>(items), 1024, 0, st>>>(a);
  } else if (vec) {
    paged_attn_whole_kernel<T, GP, LPR, true><<<static_cast<unsigned>(items), 256, 0, st>>>(a);
  }
  return check_launch("paged_attn");
}

template <typename T, int GP>
int launch_lpr(const PagedArgs& a, const Split& p, const Shape& s, bool vec, hipStream_t st) {
  switch (s.lpr) {
    case 2: return launch_paged<T, GP, 2>(a, p, s.items, vec, st);
    case 4: return launch_paged<T, GP, 4>(a, p, s.items, vec, st);
    case 8: return launch_paged<T, GP, 8>(a, p, s.items, vec, st);
    case 16: return launch_paged<T, GP, 16>(a, p, s.items, vec, st);
    case 32: return launch_paged<T, GP, 32>(a, p, s.items, vec, st);
    default:
      if constexpr (sizeof(T) == 4) return launch_paged<T, GP, 64>(a, p, s.items, vec, st);
      return fail(HYDRA_ERR_UNSUPPORTED, "paged_attn: head_dim above 256");
  }
}

template <typename T>
int launch_group(const PagedArgs& a, const Split& p, const Shape& s, bool vec, hipStream_t st) {
  switch (vec ? s.gp : 8) {
    case 1: return launch_lpr<T, 1>(a, p, s, vec, st);
    case 2: return launch_lpr<T, 2>(a, p, s, vec, st);
    case 4: return launch_lpr<T, 4>(a, p, s, vec, st);
    default: return launch_lpr<T, 8>(a, p, s, vec, st);
  }
}

// One file each instantiates it for float, bf16 and f16.
extern template int launch_group<float>(const PagedArgs&, const Split&, const Shape&, bool, hipStream_t);
extern template int launch_group<bf16>(const PagedArgs&, const Split&, const Shape&, bool, hipStream_t);
extern template int launch_group<f16>(const PagedArgs&, const Split&, const Shape&, bool, hipStream_t);

}  // namespace paged
}  // namespace hydra
