// Attention of one new token per request over a paged key-value cache, gfx950.
//
//   o[n,h] = sum_t p_t v[t, h/G],  p = softmax_t(scale q[n,h] . k[t, h/G]),
//   t < lengths[n], position t in page table[n, t / page_size].
//
// A step reads each key and value once and does 4 G flops per element pair.
// 64 requests of 16384 keys, 8/2 heads of 64, bf16 (537 MB): 100 us and 5 for the
// join, 5.1 TB/s, a large copy's rate; 8 heads to a key head of 128, 16 requests
// of 16384 keys (134 MB): 32 + 6.5 us, 3.5 TB/s, and of 256, 8 requests: 33 + 15.
// Little work does not reach it.  48 requests of up to 8192 keys, 28/4 heads of
// 16 (11 MB), take 13.6 + 4.5 us: their 828 rounds are dealt out two at a time,
// so that 414 of 768 workgroups go through two chains of table, keys, softmax
// and values, one after the other, and 354 have none; then the join is launched.
// A few keys take the launch and one such chain, 5 us.
// A wave walks its keys KT at a time:
//
//  * scores S^T = K Q^T on the matrix cores: keys are the rows of the A operand,
//    loaded from the pages in the operand's own layout (16 bytes a lane), the up
//    to GP heads of the group are columns of B (the others zero).  The order of
//    the head dimension inside an operand is free as long as K and Q agree, so
//    each lane's 16 bytes are one operand of a 16-bit type (16x16x32) and four
//    of fp32 (16x16x4, full fp32 products);
//  * the softmax keeps each head's running maximum (fp32, log2 units) in the
//    lanes of its column; the sums of one lane's keys are added up at the end;
//  * P goes through KT GP floats of LDS to the lanes that hold the rows of V,
//    which accumulate p v in fp32 with plain multiply-adds: P is never rounded,
//    V needs no transposed copy, and G multiply-adds per value stay below the
//    time its bytes take while rows are long.
//
// Pages hold 16 rows or more, so the 16 keys of an operand lie in one page and
// page ids are wave-uniform scalar loads.  An entry outside the pool counts as
// absent: its keys are not seen.  Rows past a request's length are loaded at
// most within their own page and stay out of both sums, whatever they hold.
//
// Split: the keys of all (request, key head, head block) items are laid end to
// end in rounds (one tile of KT keys per wave) and dealt out evenly to the
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
  int first;                         // item of the launch's first workgroup (whole form)
  // split form: rounds of a workgroup at least, workgroups, results
  int least, groups, cus;
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

// Most waves of a workgroup (a launch takes 4 or 8, LDS is sized for 8), and keys
// of a wave's step: 4 KB of keys and as much of values in flight.  Of 128-byte keys 32: with 16, 4 requests
// of 16384 keys take 18.8 us instead of 17.3, 32 of 3001 with 28/4 heads 31.9
// instead of 28.9; with 64, 16 of 16384 take 34.0 instead of 32.0.
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
__device__ __forceinline__ int waves() { return blockDim.x >> 6; }
// Registers: 190 with 8 heads of 256-byte keys, 215 of 512, two waves a SIMD; in
// fp32 keys above 512 bytes spill 7 (2 heads) to 54 (8 heads, whole form) of 256.
constexpr int tile_keys(int lpr) { return lpr < 4 ? 64 : (lpr <= 16 ? 32 : 16); }
template <int LPR> struct Tile { static constexpr int KT = tile_keys(LPR); };

// One step of a sum over lanes that leaves each lane half of the values: lanes
// without bit OFF keep v[0 .. N/2), the others v[N/2 .. N), to v[0 .. N/2).
template <int OFF, int N>
__device__ __forceinline__ void half_sum(float* v) {
  const bool upper = threadIdx.x & OFF;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if constexpr (OFF == 32 || OFF == 16) {
      // swaps a's upper lanes (of 64, of each 32) with b's lower ones: a + b is the sum
      const uint32_t lo = __float_as_uint(v[i]), hi = __float_as_uint(v[i + N / 2]);
      const auto r = OFF == 32 ? __builtin_amdgcn_permlane32_swap(lo, hi, false, false)
                               : __builtin_amdgcn_permlane16_swap(lo, hi, false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else {
      const float keep = upper ? v[i + N / 2] : v[i], give = upper ? v[i] : v[i + N / 2];
      v[i] = keep + __shfl_xor(give, OFF);
    }
  }
}

// v[N] of this lane summed over the lanes that differ from it in bits OFF ..
// LPR (down); returns the index of the first value left, `left` of them.
template <int OFF, int LPR, int N>
__device__ __forceinline__ int scatter_sum(float* v) {
  if constexpr (OFF < LPR) {
    return 0;
  } else if constexpr (N > 1) {
    half_sum<OFF, N>(v);
    return (threadIdx.x & OFF ? N / 2 : 0) + scatter_sum<OFF / 2, LPR, N / 2>(v);
  } else {
    v[0] += __shfl_xor(v[0], OFF);
    return scatter_sum<OFF / 2, LPR, 1>(v);
  }
}

// Pages of a wave's tile, one for each 16 keys, wave-uniform; -1: not there.
template <int NB>
__device__ __forceinline__ void tile_pages(const PagedArgs& a, const int* row, int key0, int len, int (&page)[NB]) {
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int key = __builtin_amdgcn_readfirstlane(key0 + 16 * b);
    const int p = key < len ? row[key >> a.shift] : -1;
    page[b] = static_cast<unsigned>(p) < static_cast<unsigned>(a.pages) ? p : -1;
  }
}

// One item's keys, rounds [t0, t1) (a tile per wave each): every wave's per-head
// max, sum and output in LDS, [kWaves][GP] twice and [kWaves][GP][HDP].
template <typename T, int GP, int LPR, bool VEC>
__device__ __forceinline__ void item_keys(const PagedArgs& a, int n, int h, int gb, int t0, int t1, float* sm) {
  constexpr int KT = Tile<LPR>::KT, E = Vec<T>::N, NC = LPR < 4 ? 1 : LPR / 4;
  constexpr int RPI = 64 / LPR;          // rows that one V load of the wave covers
  constexpr int NV = KT / RPI, NB = KT / 16;
  constexpr int HDP = LPR * E;           // hd rounded up
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4;  // operand row / column, 16-byte piece
  const int heads = min(GP, a.G - gb * GP);
  const int len = seen_keys(a, n), rmask = (1 << a.shift) - 1;
  const int* trow = a.table + n * a.table_rs;
  const char *kbase = a.k + h * a.k_st[1], *vbase = a.v + h * a.v_st[1];
  float* plds = sm + wave * KT * GP;
  int key0 = (t0 * waves() + wave) * KT;
  const int last = min(t1 * waves() * KT, len);
  int page[NB];
  if (key0 < last) tile_pages<NB>(a, trow, key0, len, page);
  const bool any = key0 < last;

  uint4 qf[NC];
  {
    const int head = h * a.G + gb * GP + (col < heads ? col : 0);
    const char* qrow = a.q + n * a.q_st[0] + static_cast<int64_t>(head) * a.q_st[1];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qf[c] = row_piece<T, VEC>(qrow, 4 * c + g4, a.hd);
      if (col >= heads) qf[c] = make_uint4(0, 0, 0, 0);
    }
  }
  float m = -INFINITY, l = 0.f;
  float acc[GP * E];
#pragma unroll
  for (int i = 0; i < GP * E; ++i) acc[i] = 0.f;

  const int vrow = lane / LPR, vpiece = lane % LPR;
  // a lane's place in a key block and in a value load, within a page
  const uint32_t klane = col * static_cast<uint32_t>(a.k_st[2]);
  const uint32_t vlane = (vrow & 15) * static_cast<uint32_t>(a.v_st[2]);
  for (; key0 < last; key0 += waves() * KT) {
    const bool tail = key0 + KT > len;
    uint4 kf[NB][NC];
    bool whole = true;  // every page is there
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      whole = whole && page[b] >= 0;
      const char* base = kbase + max(page[b], 0) * a.k_st[0] +
                         static_cast<int64_t>((key0 + 16 * b) & rmask) * a.k_st[2];
#pragma unroll
      for (int c = 0; c < NC; ++c) kf[b][c] = row_piece<T, VEC>(base + klane, 4 * c + g4, a.hd);
    }
    uint4 vf[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int b = i * RPI / 16;  // RPI = 32: the lower and the upper lanes' pages
      const char* base = vbase + max(page[b], 0) * a.v_st[0] +
                         static_cast<int64_t>((key0 + (RPI < 16 ? i * RPI : 16 * b)) & rmask) * a.v_st[2];
      if constexpr (RPI == 32) {
        const char* base1 = vbase + max(page[b + 1], 0) * a.v_st[0] +
                            static_cast<int64_t>((key0 + 16 * b + 16) & rmask) * a.v_st[2];
        base = vrow < 16 ? base : base1;
      }
      vf[i] = row_piece<T, VEC>(base + vlane, vpiece, a.hd);
    }
    int next[NB];
    const int key1 = key0 + waves() * KT;
    if (key1 < last) tile_pages<NB>(a, trow, key1, len, next);
    f32x4_t s[NB];
    float top = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      s[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) s[b] = mfma16<T>(kf[b][c], qf[c], s[b]);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[b][r] *= a.scale;
    }
    if (tail || !whole) {  // what is not seen: out of the scores, and 0 in v (0 x whatever lies there)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * b + 4 * g4 + r >= len || page[b] < 0) s[b][r] = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int b = i * RPI / 16;
        bool there = page[b] >= 0;
        if constexpr (RPI == 32) {
          // loaded before the choice: a chosen index would put the pages in memory
          const bool upper = page[b + 1] >= 0;
          there = vrow < 16 ? there : upper;
        }
        if (key0 + i * RPI + vrow >= len || !there) vf[i] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[b][r]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = halves_max(top);
    if (__any(top > m)) {
      const float mn = fmaxf(m, top);
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float al = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(alpha), g));
#pragma unroll
        for (int e = 0; e < E; ++e) acc[g * E + e] *= al;
      }
    }
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - ms);
        l += s[b][r];
      }
    if (col < GP) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) plds[(16 * b + 4 * g4 + r) * GP + col] = s[b][r];
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
        for (int e = 0; e < E; ++e) acc[g * E + e] = fmaf(p[g], v[e], acc[g * E + e]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int b = 0; b < NB; ++b) page[b] = next[b];
  }
  // The wave's own sums, each lane its share of the values.
  float* wm = sm;
  float* wl = sm + kWaves * GP;
  float* wa = sm + 2 * kWaves * GP;
  constexpr int ROWS = 64 / LPR, LEFT = GP * E > ROWS ? GP * E / ROWS : 1;
  int first = 0;
  if (any) {
    l += __shfl_xor(l, 16);
    l = halves_sum(l);
    first = scatter_sum<32, LPR, GP * E>(acc);
  }
  __syncthreads();  // P's memory is free
  if (lane < GP) {
    wm[wave * GP + lane] = m;
    wl[wave * GP + lane] = l;
  }
  if (any) {  // a wave without keys leaves nothing: join_waves does not look at it
#pragma unroll
    for (int i = 0; i < LEFT; ++i) {
      const int g = (first + i) / E, e = (first + i) % E;
      wa[(wave * GP + g) * HDP + vpiece * E + e] = acc[i];
    }
  }
  __syncthreads();
}

// The waves' results of item_keys as (max, sum, output element) of head g.
template <int GP, int HDP>
__device__ __forceinline__ void join_waves(const float* sm, int g, int d, float& m, float& l, float& o) {
  m = -INFINITY;
#pragma unroll 4
  for (int w = 0; w < waves(); ++w) m = fmaxf(m, sm[w * GP + g]);
  const float ms = m == -INFINITY ? 0.f : m;
  l = 0.f;
  o = 0.f;
#pragma unroll 4
  for (int w = 0; w < waves(); ++w) {
    const float mw = sm[w * GP + g], c = __builtin_amdgcn_exp2f(mw - ms);
    l = fmaf(c, sm[kWaves * GP + w * GP + g], l);
    if (mw != -INFINITY) o = fmaf(c, sm[2 * kWaves * GP + (w * GP + g) * HDP + d], o);
  }
}

template <int GP, int LPR, typename T>
constexpr int lds_floats() {
  constexpr int p = kWaves * Tile<LPR>::KT * GP, j = 2 * kWaves * GP + kWaves * GP * LPR * Vec<T>::N;
  return p > j ? p : j;
}

template <typename T>
__device__ __forceinline__ T* out_row(const PagedArgs& a, int n, int head) {
  return reinterpret_cast<T*>(a.out + n * a.o_st[0] + static_cast<int64_t>(head) * a.o_st[1]);
}

template <int LPR>
__device__ __forceinline__ int rounds_of(int len) {
  const int R = waves() * Tile<LPR>::KT;
  return len / R + (len % R != 0);
}

// The workgroup's whole item, normalised; a request without keys gets zeros.
template <typename T, int GP, int HDP>
__device__ __forceinline__ void write_out(const PagedArgs& a, int n, int h, int gb, const float* sm) {
  const int heads = min(GP, a.G - gb * GP);
  for (int e = threadIdx.x; e < heads * a.hd; e += static_cast<int>(blockDim.x)) {
    const int g = e / a.hd, d = e - g * a.hd;
    float m, l, o;
    join_waves<GP, HDP>(sm, g, d, m, l, o);
    out_row<T>(a, n, h * a.G + gb * GP + g)[d] = from_f32<T>(l == 0.f ? 0.f : o / l);
  }
}

// One workgroup per item, no split.
template <typename T, int GP, int LPR, bool VEC>
__global__ __launch_bounds__(kThreads) void paged_attn_whole_kernel(PagedArgs a) {
  constexpr int HDP = LPR * Vec<T>::N;
  __shared__ __attribute__((aligned(16))) float sm[lds_floats<GP, LPR, T>()];
  const int item = a.first + blockIdx.x, gb = item % a.GB, h = item / a.GB % a.Hkv, n = item / a.GB / a.Hkv;
  item_keys<T, GP, LPR, VEC>(a, n, h, gb, 0, rounds_of<LPR>(seen_keys(a, n)), sm);
  write_out<T, GP, HDP>(a, n, h, gb, sm);
}

// A part of an item: per-head max at 0, sum at 8, output rows from 16 on, rounded
// up to 16 bytes.
__device__ __host__ __forceinline__ int row4(int hd) { return (hd + 3) & ~3; }
template <int GP>
__device__ __forceinline__ int part_floats(int hd) { return 16 + GP * row4(hd); }

// Split form: workgroup w works on the rounds [w per, (w+1) per) of all items.
template <typename T, int GP, int LPR, bool VEC>
__global__ __launch_bounds__(kThreads) void paged_attn_split_kernel(PagedArgs a) {
  constexpr int HDP = LPR * Vec<T>::N;
  __shared__ __attribute__((aligned(16))) float sm[lds_floats<GP, LPR, T>()];
  __shared__ int pre[kMaxRequests + 1];
  __shared__ int wsum[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // prefix sums of the requests' rounds: of up to 64 requests in each wave's lanes,
  // of more in LDS
  const bool few = a.N <= 64;
  int base = 0, incl = 0;
  if (few) {
    incl = wave_incl_sum(lane < a.N ? rounds_of<LPR>(seen_keys(a, lane)) : 0);
    base = __builtin_amdgcn_readlane(incl, 63);
  } else {
    if (tid == 0) pre[0] = 0;
    for (int i0 = 0; i0 < a.N; i0 += static_cast<int>(blockDim.x)) {
      const int i = i0 + tid;
      int s = wave_incl_sum(i < a.N ? rounds_of<LPR>(seen_keys(a, i)) : 0);
      if (lane == 63) wsum[wave] = s;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < waves(); ++w) {
        if (w < wave) s += wsum[w];
        all += wsum[w];
      }
      if (i < a.N) pre[i + 1] = base + s;
      base += all;
      __syncthreads();
    }
  }
  auto before = [&](int i) {  // rounds of the requests before i, wave-uniform
    if (!few) return pre[i];
    const int s = __builtin_amdgcn_readlane(incl, max(i - 1, 0));
    return i == 0 ? 0 : s;
  };
  const int HG = a.Hkv * a.GB, total = base * HG;
  // two rounds and more, for the sake of each share's end, unless that left CUs idle
  // (4 requests of 16384 keys, 8/2 heads of 64: 17.3 us, 18.7 with single rounds)
  int per = (total + a.groups - 1) / a.groups;
  per = max(max(per, min(2, (total + a.cus - 1) / a.cus)), a.least);
  if (blockIdx.x == 0) {  // for the joining kernel
    if (tid == 0) a.plan[0] = per;
    if (few) {
      if (tid < a.N) a.plan[2 + tid] = incl;
      if (tid == 0) a.plan[1] = 0;
    } else {
      for (int i = tid; i <= a.N; i += static_cast<int>(blockDim.x)) a.plan[1 + i] = pre[i];
    }
  }
  // the last workgroup's range may pass int only if the total does (checked on the host)
  const int begin = min(static_cast<int64_t>(blockIdx.x) * per, static_cast<int64_t>(total));
  const int end = min(static_cast<int64_t>(begin) + per, static_cast<int64_t>(total));
  int n = 0;
  if (few) {  // requests that end before it
    n = __popcll(__ballot(lane < a.N && incl * HG <= begin));
  } else if (begin < end) {  // the last n with pre[n] HG <= begin
    int hi = a.N;
    while (hi - n > 1) {
      const int mid = (n + hi) >> 1;
      if (pre[mid] * HG <= begin) n = mid; else hi = mid;
    }
  }
  for (int u = begin; u < end;) {
    while (before(n + 1) * HG <= u) ++n;
    const int r = before(n + 1) - before(n), at = u - before(n) * HG, hg = at / r, t0 = at - hg * r;
    const int count = min(r - t0, end - u), h = hg / a.GB, gb = hg - h * a.GB;
    item_keys<T, GP, LPR, VEC>(a, n, h, gb, t0, t0 + count, sm);
    if (count == r) {
      write_out<T, GP, HDP>(a, n, h, gb, sm);
    } else {
      float* part = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (u == begin ? 0 : 1)) * part_floats<GP>(a.hd);
      for (int e = tid; e < GP * a.hd; e += static_cast<int>(blockDim.x)) {
        const int g = e / a.hd, d = e - g * a.hd;
        float m, l, o;
        join_waves<GP, HDP>(sm, g, d, m, l, o);
        part[16 + g * row4(a.hd) + d] = o;
        if (d == 0) {
          part[g] = m;
          part[8 + g] = l;
        }
      }
    }
    u += count;
    __syncthreads();
  }
}

// Joins the parts of one item, in their order; writes the zeros of a request
// without keys.  Items that one workgroup had whole are written already.
// Four elements a thread, the parts dealt out over the threads left, eight loads
// of 16 bytes in flight each.
template <typename T, int GP>
__global__ __launch_bounds__(1024) void paged_attn_join_kernel(PagedArgs a) {
  constexpr int PL = kMaxParts / 64;
  __shared__ float weight[GP][kMaxParts];
  __shared__ float4 sums[1024];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int HG = a.Hkv * a.GB, n = blockIdx.x / HG, hg = blockIdx.x - n * HG, h = hg / a.GB, gb = hg - h * a.GB;
  const int per = a.plan[0], p0 = a.plan[1 + n], r = a.plan[2 + n] - p0;
  const int heads = min(GP, a.G - gb * GP);
  const int u0 = p0 * HG + hg * r, w0 = u0 / per, parts = r == 0 ? 0 : (u0 + r - 1) / per - w0 + 1;
  if (parts == 1) return;
  auto part = [&](int p) {  // only the first one can begin inside its workgroup's range
    return a.part + (static_cast<int64_t>(w0 + p) * 2 + (p == 0 && u0 != w0 * per ? 1 : 0)) * part_floats<GP>(a.hd);
  };
  for (int g = wave; g < GP; g += 16) {
    float m[PL], l[PL], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const int p = lane + 64 * i;
      m[i] = p < parts ? part(p)[g] : -INFINITY;
      l[i] = p < parts ? part(p)[8 + g] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < PL; ++i) top = fmaxf(top, m[i]);
    top = wave_max(top);
    const float ts = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      m[i] = __builtin_amdgcn_exp2f(m[i] - ts);
      sum = fmaf(m[i], l[i], sum);
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < PL; ++i) weight[g][lane + 64 * i] = m[i] * inv;
  }
  __syncthreads();
  const int quads = row4(a.hd) / 4, elems = heads * quads;
  int lanes = 1;  // threads of four elements
  while (lanes < 64 && lanes * 2 * elems <= 1024) lanes *= 2;
  const int step = 1024 / lanes, sub = tid / step;
  for (int e0 = 0; e0 < elems; e0 += step) {
    const int e = e0 + tid - sub * step;
    const int g = e < elems ? e / quads : 0, d = 4 * (e - g * quads);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e < elems) {
      for (int p = sub; p < parts; p += 8 * lanes) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int q = min(p + j * lanes, parts - 1);
          const float c = weight[g][q];
          const float4 x = *reinterpret_cast<const float4*>(part(q) + 16 + g * row4(a.hd) + d);
          // by its number, not by its weight: 0 x NaN of a part whose weight vanishes is NaN
          if (p + j * lanes < parts) {
            o.x = fmaf(c, x.x, o.x);
            o.y = fmaf(c, x.y, o.y);
            o.z = fmaf(c, x.z, o.z);
            o.w = fmaf(c, x.w, o.w);
          }
        }
      }
    }
    sums[tid] = o;
    __syncthreads();
    if (sub == 0 && e < elems) {
      for (int i = 1; i < lanes; ++i) {
        const float4 x = sums[i * step + tid];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
      }
      T* out = out_row<T>(a, n, h * a.G + gb * GP + g) + d;
      const float v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < a.hd) out[i] = from_f32<T>(v[i]);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------- launch
struct Shape {
  int gp, lpr, kt, row;  // row: bytes of a key
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
  s.row = static_cast<int>(hd) * e;
  s.items = N * Hkv * s.gb;
  return s;
}

struct Split {
  bool on;
  int least, waves;
};

constexpr int kMaxResident = 4;  // workgroups of a CU that a split launch takes at most (8: the same times)

// Split where the items alone would not fill the chip and a request may be longer
// than 128 KB of keys or 2048 of them, whole and split with its join: of 128-byte
// keys 512 take 8.0 and 10.3 us, 1000 10.5 and 10.6, 2000 15.6 and 10.8; of 32-byte
// keys 2000 take 9.9 and 11.0, 4000 15.1 and 11.1.  8 waves for few short items (one request of
// 500 keys, 28/4 heads of 64: 9.4 us, 11.4 with 4); where items or rounds are many,
// twice as many workgroups of 4 have more of the chip's registers in use (256
// requests of 20 keys, 28/4 heads of 64: 8.0 us, 11.8 with 8).
inline Split split_of(const Shape& s, int64_t N, int64_t capacity) {
  Split r{};
  r.on = N <= kMaxRequests && s.items < 8 * device_cus() && capacity > std::min<int64_t>(2048, (128 << 10) / s.row);
  r.waves = r.on || s.items > device_cus() ? 4 : kWaves;
  const int64_t most = (capacity + r.waves * s.kt - 1) / (r.waves * s.kt);
  r.on = r.on && most * s.items < (int64_t(1) << 31) - (1 << 20);  // rounds and workgroups in an int
  r.least = static_cast<int>(std::max<int64_t>(1, (most + kMaxParts - 2) / (kMaxParts - 1)));
  return r;
}

// The plan's whole numbers, rounded up to 16 bytes.
inline int64_t plan_ints(int64_t N) { return (N + 2 + 3) / 4 * 4; }

inline int64_t workspace_bytes(const Split& p, int64_t N, int64_t hd) {
  if (!p.on) return 0;
  const int64_t parts = static_cast<int64_t>(kMaxResident) * device_cus() * 2;
  return 4 * (plan_ints(N) + parts * (16 + 8 * row4(static_cast<int>(hd))));
}

template <typename T, int GP, int LPR, bool VEC>
void launch_form(PagedArgs a, const Split& p, int64_t items, hipStream_t st) {
  if (p.on) {
    // as many workgroups as are resident at once, which the rounds are dealt to
    const auto kernel = paged_attn_split_kernel<T, GP, LPR, VEC>;
    a.cus = device_cus();
    a.groups = a.cus * std::min(kMaxResident, blocks_per_cu(reinterpret_cast<const void*>(kernel), 64 * p.waves));
    kernel<<<a.groups, 64 * p.waves, 0, st>>>(a);
  } else {
    // HIP counts a launch's threads in 32 bits
    constexpr int64_t most = int64_t(1) << 22;
    for (int64_t first = 0; first < items; first += most) {
      a.first = static_cast<int>(first);
      paged_attn_whole_kernel<T, GP, LPR, VEC>
          <<<static_cast<unsigned>(std::min(most, items - first)), 64 * p.waves, 0, st>>>(a);
    }
  }
}

// Rows that 16-byte loads cannot take come through one form, of 8 heads.
template <typename T, int GP, int LPR>
int launch_paged(const PagedArgs& a, const Split& p, int64_t items, bool vec, hipStream_t st) {
  if constexpr (GP == 8) {
    if (!vec) launch_form<T, GP, LPR, false>(a, p, items, st);
  }
  if (vec) launch_form<T, GP, LPR, true>(a, p, items, st);
  if (p.on) paged_attn_join_kernel<T, GP><<<static_cast<unsigned>(items), 1024, 0, st>>>(a);
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
