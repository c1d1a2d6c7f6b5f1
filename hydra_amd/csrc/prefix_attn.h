// Attention of one new token per request over a paged key-value cache whose
// pages hold 8 bits, or whose requests share a prefix in groups, gfx950.
//
//   o[n,h] = sum_t p_t v[t, h/G],  p = softmax_t(scale q[n,h] . k[t, h/G]),
//   t < lengths[n], position t in page table[n, t / page_size];
//   in 8 bits k[t] = ks[t] K[t] and v[t] = vs[t] V[t], a scale for each row.
//
// Requests come in groups of W.  The first shared[g] positions of group g are
// the same for all of its requests that are as long: their keys and values are
// read once, as one product of W G rows, and each request's own positions behind
// them (from the last whole 16 on) by themselves.  Both are *items* of one
// kind, a set of query rows and a range of keys of one table row:
//
//   A  (group, key head, block of rows): up to 32 rows a workgroup where the
//      group has no more (its waves take the keys in turn), else 128 (each wave
//      32 rows of its own, all waves the same keys); in the form of 256 channels,
//      and in fp32 in that of 128, up to 16, else 64 (16 a wave);
//   B  (request, key head, block of 16 heads): the waves take the keys in turn.
//
// A wave walks its keys 32 at a time, on the matrix cores throughout:
//
//  * scores S^T = K Q^T, 16 keys by 16 rows: the keys are loaded from the pages
//    in the operand's own layout (16 bytes a lane; the order of the head
//    dimension inside an operand is free as long as K and Q agree).  8 bits
//    become bf16 (of fp16 queries fp16, of fp32 ones fp32), which hold them
//    exactly; ks goes into the score in fp32;
//  * the softmax keeps each row's running maximum and sum in fp32 in the lanes
//    of its column;
//  * O^T = V^T P^T: the lanes' scores are the operand's layout already.  V is
//    staged through LDS, whose transposing read gives its columns.  P vs is
//    taken as two 16-bit terms, its rounding and what that leaves: 2^-16 of it in
//    bf16 (2^-22 in fp16), so that the result is rounded once, in effect.  It
//    costs a second matrix instruction where the softmax's arithmetic is the
//    longer part.  fp16's least step is 2^-24, which many light weights beside a heavy
//    one are all below: they enter times 2^15 (2^13 where the maximum lags behind), so
//    that of each at most 2^-38 of the largest weight is lost.  In fp32 all operands
//    are fp32.
//
// Split: A items are cut into pieces of whole rounds (128 keys), one to a workgroup
// where they suffice; the rounds of all B items are laid end to end and dealt out to
// all workgroups so that each has as much to do, whatever the lengths.  What a workgroup leaves of an item is (max, sum, unscaled
// output) per row in the workspace; a second kernel joins each row's parts in their
// order.  No atomics on results: the same inputs give the same bits.
//
// What bounds it, by the kernels' own times:
//
//  * B items, many long ones: the reading of the pages.  64 requests of 16384 keys, 8/2
//    heads of 64 in e4m3 (285 MB) take 53.8 us, 5.3 TB/s, and 4.9 us to join; 256 of
//    4096, 32/8 heads of 128 in int8 (2.2 GB), 386 us, 5.7 TB/s.  For fp32 queries it is
//    the fp32 products, of 16 rows of which these heads fill 4: 109 and 786 us;
//  * A items of many rows: the matrix cores and the softmax, in turn.  256 requests that
//    share 32768 keys, 32/8 heads of 128 (137 GFLOP), with 600 keys of their own each:
//    227 to 251 us, as the clock goes (over e4m3 334, int8 372: their general form widens
//    every tile of keys in each wave; once for all of them, through LDS, it was 336 and
//    355).  The products, 206 GFLOP with the second terms of P, and their operands' reads
//    from LDS take 160 us with all else left out, the rate of a large library product;
//    without the second terms the whole takes 36 us less, without the softmax 36, without
//    the loads 16.  With 256 channels 717 us (over e4m3 1056), one workgroup to a CU;
//  * the same in fp32, 4096 shared keys: the fp32 products, 330 us of 112 at 128 channels,
//    where one workgroup a CU fits, 895 of 223 at 256, where registers are spilt;
//  * few requests: the chain of launch, plan, table, keys and join.  8 groups of 4
//    requests by 1500 keys: 8.4 us and 4.3 to join; one request of 700: 8.6 us.
#pragma once
#include "common.h"
#include "lds_dma.h"
#include "mod_keys.h"

#include <algorithm>
#include <type_traits>

namespace hydra {
namespace prefix {

struct i8 { int8_t bits; };
struct e4m3 { uint8_t bits; };

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRequests = 1024;  // of one launch: prefix sums of their rounds lie in LDS
constexpr int kRound = 128;      // keys
constexpr int kThreads = 256;

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;

struct PrefixArgs {
  const char *q, *k, *v;
  char* out;
  const float *ks, *vs;         // scales of 8-bit rows
  int64_t q_st[2], o_st[2];     // bytes: n, h
  int64_t k_st[3], v_st[3];     // bytes: page, h, row
  int64_t ks_st[2], vs_st[2];   // elements: page, h
  const int *table, *lengths, *shared;  // shared: null without groups
  int64_t table_rs;
  int N, H, Hkv, hd, G, W, groups, P, shift, pages;
  int GB, RB;                   // blocks of 16 heads, of A rows
  float scale;                  // times log2(e)
  bool split;                   // else one workgroup of `waves` takes one B item, `first` and on
  int waves, first, wgs, cus;
  int* plan;                    // see kPlan
  float* part;                  // slots: pieces of A, then [wgs][2] of B, then (with groups) whole B items
  int64_t slot_a, slot_b, part_b, whole_b;  // floats of a slot, offsets in part
};

// The plan's whole numbers: how B is dealt out (Deal), then prefix sums of the groups'
// pieces and of the requests' rounds.
enum { kWgsA, kBeside, kPer, kPlan };

// What depends on the type of the pages and of the queries.
template <typename C, typename KV> struct Types {
  static constexpr bool eight = sizeof(KV) == 1;
  static constexpr bool f32 = sizeof(C) == 4;
  using VT = std::conditional_t<f32, float, std::conditional_t<eight, bf16, C>>;  // V in LDS, and P
  static constexpr bool f16_p = std::is_same<VT, f16>::value;
};

constexpr int pitch_of(int hdp, bool f32) { return f32 ? hdp + 4 : (hdp == 32 || hdp == 128 ? hdp + 16 : hdp + 8); }
constexpr int tile_keys(int hdp, bool f32) { return f32 && hdp == 256 ? 16 : 32; }
constexpr int tiles_a(int hdp, bool f32) { return hdp == 256 || (f32 && hdp == 128) ? 1 : 2; }  // of 16 rows, a wave

template <typename T>
__device__ __forceinline__ f32x4_t mfma32(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}

// Four 8-bit values of a word, exactly, as two words of a 16-bit type or as fp32.
template <typename KV, typename T>
__device__ __forceinline__ uint2 widen(uint32_t w) {
  if constexpr (std::is_same<KV, e4m3>::value) {
    if constexpr (std::is_same<T, bf16>::value)
      return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)));
    else
      return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)));
  } else {
    const int s = static_cast<int>(w);
    const float a = static_cast<float>(static_cast<int8_t>(s)), b = static_cast<float>(static_cast<int8_t>(s >> 8));
    const float c = static_cast<float>(static_cast<int8_t>(s >> 16)), d = static_cast<float>(s >> 24);
    return make_uint2(pack2<T>(a, b), pack2<T>(c, d));
  }
}
template <typename KV>
__device__ __forceinline__ float4 widen_f32(uint32_t w) {
  if constexpr (std::is_same<KV, e4m3>::value) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return make_float4(lo[0], lo[1], hi[0], hi[1]);
  } else {
    const int s = static_cast<int>(w);
    return make_float4(static_cast<float>(static_cast<int8_t>(s)), static_cast<float>(static_cast<int8_t>(s >> 8)),
                       static_cast<float>(static_cast<int8_t>(s >> 16)), static_cast<float>(s >> 24));
  }
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Piece `piece` (16 bytes) of a row of hd elements of T; zeros past its end.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 row_piece(const char* row, int piece, int hd) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (VEC) {
    return piece * E < hd ? *reinterpret_cast<const uint4*>(row + piece * 16) : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = piece * E + i;
      uint32_t x = 0;
      if (e < hd) {
        const char* p = row + e * static_cast<int>(sizeof(T));
        if constexpr (sizeof(T) == 1) x = *reinterpret_cast<const uint8_t*>(p);
        else if constexpr (sizeof(T) == 2) x = *reinterpret_cast<const uint16_t*>(p);
        else x = *reinterpret_cast<const uint32_t*>(p);
      }
      w[i * static_cast<int>(sizeof(T)) / 4] |= x << (i * 8 * static_cast<int>(sizeof(T)) % 32);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The weights of 8 keys as two operands of a 16-bit type: rounded, and what that leaves.
template <typename T>
__device__ __forceinline__ void two_terms(const f32x4_t& a, const f32x4_t& b, uint4& hi, uint4& lo) {
  uint32_t h[4], x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float p0 = i < 2 ? a[2 * i] : b[2 * i - 4], p1 = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
    h[i] = pack2<T>(p0, p1);
    if constexpr (std::is_same<T, bf16>::value) {
      asm("" : "+v"(h[i]));  // one conversion of the pair: the compiler would make three of it
      x[i] = pack2<T>(p0 - __uint_as_float(h[i] << 16), p1 - __uint_as_float(h[i] & 0xffff0000u));
    } else {
      const f16x2_t w = __builtin_bit_cast(f16x2_t, h[i]);
      x[i] = pack2<T>(p0 - static_cast<float>(w[0]), p1 - static_cast<float>(w[1]));
    }
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(x[0], x[1], x[2], x[3]);
}

// Four scales of neighbouring rows.
template <bool VEC>
__device__ __forceinline__ f32x4_t four_scales(const float* p) {
  if constexpr (VEC) return *reinterpret_cast<const f32x4_t*>(p);
  return f32x4_t{p[0], p[1], p[2], p[3]};
}

__device__ __forceinline__ int clamp_len(const PrefixArgs& a, int len) { return max(0, min(len, a.P << a.shift)); }
// Positions of group g that are read once, whole 16s.
__device__ __forceinline__ int shared_keys(const PrefixArgs& a, int g) {
  return a.shared ? clamp_len(a, a.shared[g]) & ~15 : 0;
}

// Rows row0 .. of an item: request n0 + r / G, head h G + r % G.  Keys
// [begin, end) of table row `trow`, whose requests all see them.
struct Item {
  int n0, h, row0, rows;  // rows: of the item from row0 on, at most the workgroup's
  int trow, begin, end;
};

// The same in scalar registers: what prefix sums in LDS gave counts as different in
// each lane, and pages would be looked up by vector loads in line with the keys'.
__device__ __forceinline__ Item uniform(const Item& i) {
  auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return Item{u(i.n0), u(i.h), u(i.row0), u(i.rows), u(i.trow), u(i.begin), u(i.end)};
}

// A wave's state of NT tiles of 16 rows: lane = column (row of the item) and group of four.
template <int HDP, int NT> struct State {
  f32x4_t o[NT][HDP / 16];
  float m[NT], l[NT];
};

// Pages of a tile, one for each 16 keys, wave-uniform (scalar loads: nothing in the
// launch writes the table); -1: not there.
__device__ __forceinline__ int page_of(const PrefixArgs& a, const int* row, int key0, int end) {
  typedef const __attribute__((address_space(4))) int* const_t;
  const const_t at = (const_t)(reinterpret_cast<uintptr_t>(row));
  const int key = __builtin_amdgcn_readfirstlane(key0);
  const int p = key < end ? at[key >> a.shift] : -1;
  return static_cast<unsigned>(p) < static_cast<unsigned>(a.pages) ? p : -1;
}
template <int NB>
__device__ __forceinline__ void tile_pages(const PrefixArgs& a, const int* row, int key0, int end, int (&page)[NB]) {
#pragma unroll
  for (int b = 0; b < NB; ++b) page[b] = page_of(a, row, key0 + 16 * b, end);
}

// An item's keys.  RW = 1: the NW waves take tiles in turn, and wave 0 ends up with
// all of their sums; RW = 4: each wave has rows of its own.
template <typename C, typename KV, int HDP, int NT, int RW, bool VEC, int NW = 4>
__device__ __forceinline__ void item_keys(const PrefixArgs& a, const Item& item, char* lds, State<HDP, NT>& st) {
  const Item it = uniform(item);
  using Ty = Types<C, KV>;
  using VT = typename Ty::VT;
  constexpr bool F32 = Ty::f32, EIGHT = Ty::eight;
  constexpr float LIFT = Ty::f16_p ? 15.f : 0.f;  // of the weights' exponents, which are at most 0
  constexpr int KT = tile_keys(HDP, F32), NB = KT / 16, KW = NW / RW, TT = 64 * RW;
  constexpr int E = 16 / sizeof(KV);                       // elements of a piece
  constexpr int PPR = HDP / E > 0 ? HDP / E : 1;           // pieces of a row
  constexpr int NC = PPR < 4 ? 1 : PPR / 4;                // pieces of a lane
  constexpr int NV = KT * PPR <= TT ? 1 : KT * PPR / TT;   // V pieces of a thread
  constexpr int QE = NC * E;                               // q elements of a lane
  constexpr int PITCH = pitch_of(HDP, F32), TILE = KT * PITCH * static_cast<int>(sizeof(VT));
  constexpr int NO = HDP / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int kw = RW == 1 ? wave : 0, tt = RW == 1 ? lane : tid;
  const int rmask = (1 << a.shift) - 1;
  const int* trow = a.table + it.trow * a.table_rs;
  const char *kbase = a.k + it.h * a.k_st[1], *vbase = a.v + it.h * a.v_st[1];
  const float *ksb = EIGHT ? a.ks + it.h * a.ks_st[1] : nullptr, *vsb = EIGHT ? a.vs + it.h * a.vs_st[1] : nullptr;
  char* tile = lds + (RW == 1 ? wave * TILE : 0);

  // q, in the order of the keys' pieces; rows that are none: zeros
  uint4 qf[NT][QE * sizeof(C) / 16];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (RW == 1 ? 0 : wave * 16 * NT) + 16 * t + col;
    const bool there = r < it.rows;
    const int at = it.row0 + (there ? r : 0), n = it.n0 + at / a.G, head = it.h * a.G + at % a.G;
    const char* qrow = a.q + n * a.q_st[0] + static_cast<int64_t>(head) * a.q_st[1];
    constexpr int PQ = E * sizeof(C) / 16;  // q pieces beside one of the keys'
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < PQ; ++j) {
        uint4 x = row_piece<C, VEC>(qrow, (4 * c + g4) * PQ + j, a.hd);
        if (!there) x = make_uint4(0, 0, 0, 0);
        qf[t][c * PQ + j] = x;
      }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    st.m[t] = -INFINITY;
    st.l[t] = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i) st.o[t][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  int key0 = it.begin + kw * KT;
  const uint32_t klane = col * static_cast<uint32_t>(a.k_st[2]);
  int vrow[NV], vpiece[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = i * TT + tt;
    vrow[i] = e / PPR;
    vpiece[i] = e % PPR;
  }
  int page[NB], next[NB];
  uint4 kf[NB][NC], vf[NV];
  f32x4_t ksf[NB], vsf[NB];
  auto load_v = [&](const int (&pg)[NB], int k0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int b = vrow[i] >> 4;
      int p = pg[0];
#pragma unroll
      for (int x = 1; x < NB; ++x) p = b == x ? pg[x] : p;
      const bool in = KT * PPR >= TT || vrow[i] < KT;
      const char* base = vbase + max(p, 0) * a.v_st[0] + static_cast<int64_t>((k0 + 16 * (b < NB ? b : 0)) & rmask) * a.v_st[2] +
                         (vrow[i] & 15) * static_cast<uint32_t>(a.v_st[2]);
      vf[i] = in ? row_piece<KV, VEC>(base, vpiece[i], a.hd) : make_uint4(0, 0, 0, 0);
    }
  };
  auto load_k = [&](const int (&pg)[NB], int k0) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int64_t p = max(pg[b], 0);
      const int r = (k0 + 16 * b) & rmask;
      const char* base = kbase + p * a.k_st[0] + static_cast<int64_t>(r) * a.k_st[2];
#pragma unroll
      for (int c = 0; c < NC; ++c) kf[b][c] = row_piece<KV, VEC>(base + klane, 4 * c + g4, a.hd);
      if constexpr (EIGHT) {
        ksf[b] = four_scales<VEC>(ksb + p * a.ks_st[0] + r + 4 * g4);
        vsf[b] = four_scales<VEC>(vsb + p * a.vs_st[0] + r + 4 * g4);
      }
    }
  };
  if (key0 < it.end) {
    tile_pages<NB>(a, trow, key0, it.end, page);
    load_v(page, key0);
    load_k(page, key0);
    tile_pages<NB>(a, trow, key0 + KW * KT, it.end, next);
  }
  int turn = 0;
  for (; key0 < it.end; key0 += KW * KT) {
    const int key1 = key0 + KW * KT;
    bool whole = key0 + KT <= it.end;  // all keys are there
#pragma unroll
    for (int b = 0; b < NB; ++b) whole = whole && page[b] >= 0;
    VT* vt = reinterpret_cast<VT*>(RW == 1 ? tile : lds + (turn & 1) * TILE);
    turn ^= 1;
    // V into LDS; rows that are not seen as zeros (0 x whatever lies there)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (KT * PPR < TT && vrow[i] >= KT) continue;
      if (!whole) {
        int p = page[0];
#pragma unroll
        for (int x = 1; x < NB; ++x) p = (vrow[i] >> 4) == x ? page[x] : p;
        if (key0 + vrow[i] >= it.end || p < 0) vf[i] = make_uint4(0, 0, 0, 0);
      }
      VT* to = vt + vrow[i] * PITCH + vpiece[i] * E;
      if constexpr (!EIGHT) {
        *reinterpret_cast<uint4*>(to) = vf[i];
      } else if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(to + 4 * j) = widen_f32<KV>(word(vf[i], j));
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint2 x = widen<KV, VT>(word(vf[i], 2 * j)), y = widen<KV, VT>(word(vf[i], 2 * j + 1));
          *reinterpret_cast<uint4*>(to + 8 * j) = make_uint4(x.x, x.y, y.x, y.y);
        }
      }
    }
    if (key1 < it.end) load_v(next, key1);
    // scores
    f32x4_t s[NB][NT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < NT; ++t) s[b][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (F32) {
          float x[E];
          if constexpr (EIGHT) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 f = widen_f32<KV>(word(kf[b][c], j));
              x[4 * j] = f.x, x[4 * j + 1] = f.y, x[4 * j + 2] = f.z, x[4 * j + 3] = f.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(word(kf[b][c], j));
          }
#pragma unroll
          for (int j = 0; j < E; ++j)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              s[b][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  x[j], __uint_as_float(word(qf[t][(c * E + j) / 4], j & 3)), s[b][t], 0, 0, 0);
        } else if constexpr (EIGHT) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint2 x = widen<KV, C>(word(kf[b][c], 2 * j)), y = widen<KV, C>(word(kf[b][c], 2 * j + 1));
            const uint4 kk = make_uint4(x.x, x.y, y.x, y.y);
#pragma unroll
            for (int t = 0; t < NT; ++t) s[b][t] = mfma32<C>(kk, qf[t][2 * c + j], s[b][t]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < NT; ++t) s[b][t] = mfma32<C>(kf[b][c], qf[t][c], s[b][t]);
        }
      }
    f32x4_t vs[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x4_t f = {a.scale, a.scale, a.scale, a.scale};
      if constexpr (EIGHT) {
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] *= ksf[b][r];
        vs[b] = vsf[b];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][t][r] *= f[r];
    }
    if (!whole) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * b + 4 * g4 + r >= it.end || page[b] < 0) {
            vs[b][r] = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t) s[b][t][r] = -INFINITY;
          }
    }
    if (key1 < it.end) load_k(next, key1);
#pragma unroll
    for (int b = 0; b < NB; ++b) page[b] = next[b];
    if (key1 < it.end) tile_pages<NB>(a, trow, key1 + KW * KT, it.end, next);
    // softmax
    uint4 hi[NT], lo[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[b][t][r]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = halves_max(top);
      if (__any(top > st.m[t])) {
        const float mn = fmaxf(st.m[t], top);
        const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m[t] - mn);
        st.m[t] = mn;
        st.l[t] *= alpha;
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) st.o[t][i][r] *= alpha;
      }
      const float ms = st.m[t] == -INFINITY ? 0.f : st.m[t] - LIFT;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(s[b][t][r] - ms);
          st.l[t] += p;
          s[b][t][r] = EIGHT ? p * vs[b][r] : p;
        }
      if constexpr (!F32) two_terms<VT>(s[0][t], s[1][t], hi[t], lo[t]);
    }
    if constexpr (RW == 1) {  // the tile is this wave's alone; its LDS operations keep their order
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();  // two tiles in turn: the one read before this one is written after it
    }
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      if constexpr (F32) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = vt[(16 * b + 4 * g4 + r) * PITCH + 16 * i + col];
#pragma unroll
            for (int t = 0; t < NT; ++t) st.o[t][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[b][t][r], st.o[t][i], 0, 0, 0);
          }
      } else {
        // 16 lanes read 4 rows of 16 columns, lane j gets column j's four values
        typedef __attribute__((address_space(3))) s16x4_t* lds_t;
        const VT* p = vt + (4 * g4 + (col >> 2)) * PITCH + 16 * i + 4 * (col & 3);
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p)));
        const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + 16 * PITCH)));
        const uint4 vv = make_uint4(x.x, x.y, y.x, y.y);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          st.o[t][i] = mfma32<VT>(vv, hi[t], st.o[t][i]);
          st.o[t][i] = mfma32<VT>(vv, lo[t], st.o[t][i]);
        }
      }
    }
    if constexpr (RW == 1) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    st.l[t] += __shfl_xor(st.l[t], 16);
    st.l[t] = halves_sum(st.l[t]);
    if (st.m[t] != -INFINITY) st.m[t] -= LIFT;
  }
  if constexpr (RW == 1) {  // the upper half of the waves into the lower one, until one is left: all hold the same layout
    float* sm = reinterpret_cast<float*>(lds);
    constexpr int ROW = NT * (2 + 4 * NO);
#pragma unroll
    for (int half = NW / 2; half > 0; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
        float* to = sm + (wave - half) * ROW * 64 + lane;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          to[64 * (2 * t)] = st.m[t];
          to[64 * (2 * t + 1)] = st.l[t];
#pragma unroll
          for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) to[64 * (2 * NT + (t * NO + i) * 4 + r)] = st.o[t][i][r];
        }
      }
      __syncthreads();
      if (wave < half) {
        const float* from = sm + wave * ROW * 64 + lane;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float m1 = from[64 * (2 * t)], mn = fmaxf(st.m[t], m1), ms = mn == -INFINITY ? 0.f : mn;
          const float c0 = __builtin_amdgcn_exp2f(st.m[t] - ms), c1 = __builtin_amdgcn_exp2f(m1 - ms);
          st.m[t] = mn;
          st.l[t] = fmaf(c0, st.l[t], c1 * from[64 * (2 * t + 1)]);
#pragma unroll
          for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              st.o[t][i][r] = fmaf(c0, st.o[t][i][r], c1 * from[64 * (2 * NT + (t * NO + i) * 4 + r)]);
        }
      }
    }
  }
  __syncthreads();  // the LDS is free
}

// An A item of more rows than a wave takes, over pages of the queries' 16-bit type:
// the same product, with keys and values both staged in LDS by direct loads, 64 keys
// (of more than 128 channels 32) at a time and the next tile's in flight meanwhile.
// The loads write 16 bytes a lane one after the other, so it is the lanes' sources that
// are permuted: piece c of row r lies at c ^ f(r), which spreads both the rows' 16-byte
// reads (16 rows at once) and the transposing ones (8 rows of 32 bytes) over all banks.
// An item's keys end at a whole 16, so what is not seen are whole blocks of 16: their
// loads' descriptors are empty, which gives zeros.
constexpr int rows_tile(int hdp) { return hdp == 256 ? 32 : 64; }

template <typename C, int HDP, int NT>
__device__ __forceinline__ void item_rows(const PrefixArgs& a, const Item& item, char* lds, State<HDP, NT>& st) {
  const Item it = uniform(item);
  constexpr int KT = rows_tile(HDP), NB = KT / 16, PPR = HDP / 8, RPI = 64 / PPR, NJ = KT * PPR / 256;
  constexpr int NC = HDP / 32, NO = HDP / 16, TILE = KT * HDP * 2;
  constexpr int RPB = PPR < 16 ? 16 / PPR : 1, PX = PPR < 16 ? PPR : 16;  // rows of 256 bytes; pieces to permute
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4, rmask = (1 << a.shift) - 1;
  const int* trow = a.table + it.trow * a.table_rs;
  const char *kbase = a.k + it.h * a.k_st[1], *vbase = a.v + it.h * a.v_st[1];
  auto fk = [](int r) { return r / RPB % PX; };
  auto fv = [](int r) { return r / RPB % (PX / 2) * 2; };

  // q times the scale's sign: the score's product with |scale| is then monotone
  const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
  // a scale of 0 as the least normal one: scores of 0, and -inf where a key is not seen (a
  // maximum would let go of a scale that is NaN)
  const float scale = fabsf(a.scale) < 0x1p-126f ? 0x1p-126f : fabsf(a.scale);
  uint4 qf[NT][NC];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = wave * 16 * NT + 16 * t + col;
    const bool there = r < it.rows;
    const int at = it.row0 + (there ? r : 0), n = it.n0 + at / a.G, head = it.h * a.G + at % a.G;
    const char* qrow = a.q + n * a.q_st[0] + static_cast<int64_t>(head) * a.q_st[1];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint4 x = row_piece<C, true>(qrow, 4 * c + g4, a.hd);
      x = make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
      qf[t][c] = there ? x : make_uint4(0, 0, 0, 0);
    }
    st.m[t] = -INFINITY;
    st.l[t] = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i) st.o[t][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // The reference of the weights: m times the scale, 0 before the first key, less LIFT.  In
  // fp16 they are lifted, and the reference lags less behind, so that light ones stay above its
  // least step and the heaviest, 2^(LIFT + LAG), within its range.
  constexpr float LIFT = std::is_same<C, f16>::value ? 13.f : 0.f, LAG = std::is_same<C, f16>::value ? 2.f : 8.f;
  float ms[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) ms[t] = -LIFT;

  // A tile lies in one page, or its blocks of 16 may lie in several: a descriptor for the
  // tile, or for each load (which none goes beyond).
  const bool one = (KT - 1) >> a.shift == 0;
  // this lane's piece of each direct load, in the tile or in its block
  uint32_t koff[NJ], voff[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = (j * 4 + wave) * RPI + lane / PPR, c = lane % PPR, in = one ? r : r & 15;
    const uint32_t ck = c ^ fk(r), cv = c ^ fv(r), none = 0x7ffffff0u;
    koff[j] = static_cast<int>(ck) * 8 < a.hd ? in * static_cast<uint32_t>(a.k_st[2]) + 16 * ck : none;
    voff[j] = static_cast<int>(cv) * 8 < a.hd ? in * static_cast<uint32_t>(a.v_st[2]) + 16 * cv : none;
  }
  const int krow = static_cast<int>(a.k_st[2]), vrow = static_cast<int>(a.v_st[2]);
  const uint32_t base = lds_addr(lds);
  // Pages of 64 blocks of 16 keys at a time, one to a lane: looked up tile by tile they
  // would be waited for together with the operands from LDS.
  constexpr int TPB = 64 / NB;  // tiles of such a batch
  auto batch = [&](int first) {
    const int key = first + 16 * lane;
    const int p = key < it.end ? trow[key >> a.shift] : -1;
    return static_cast<unsigned>(p) < static_cast<unsigned>(a.pages) ? p : -1;
  };
  auto page_at = [](int pages, int i) { return __builtin_amdgcn_readlane(pages, i); };
  auto issue = [&](int pages, int at, int k0, int buf) {  // the batch's blocks from `at` on
    const uint32_t to = base + buf * 2 * TILE + wave * 1024;
    if (one) {
      const int p = page_at(pages, at), rows = min(KT, it.end - k0);
      const int64_t r = k0 & rmask, pg = max(p, 0);
      const i32x4_t ks = raw_rsrc(kbase + pg * a.k_st[0] + r * krow, p < 0 ? 0 : (rows - 1) * krow + 2 * a.hd);
      const i32x4_t vs = raw_rsrc(vbase + pg * a.v_st[0] + r * vrow, p < 0 ? 0 : (rows - 1) * vrow + 2 * a.hd);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        load16_to_lds(ks, to + j * 4096, koff[j]);
        load16_to_lds(vs, to + j * 4096 + TILE, voff[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int b = (j * 4 + wave) * RPI >> 4, p = page_at(pages, at + b);
        const int64_t r = (k0 + 16 * b) & rmask, pg = max(p, 0);
        load16_to_lds(raw_rsrc(kbase + pg * a.k_st[0] + r * krow, p < 0 ? 0 : 15 * krow + 2 * a.hd), to + j * 4096, koff[j]);
        load16_to_lds(raw_rsrc(vbase + pg * a.v_st[0] + r * vrow, p < 0 ? 0 : 15 * vrow + 2 * a.hd), to + j * 4096 + TILE,
                      voff[j]);
      }
    }
  };
  const uint32_t kread = col * HDP * 2 + ((g4 ^ fk(col)) << 4);
  const int vr = 4 * g4 + (col >> 2);
  const uint32_t vread = vr * HDP * 2 + ((((col & 3) >> 1) ^ fv(vr)) << 4) + (col & 1) * 8;

  int pages = batch(it.begin), next = -1;
  __builtin_amdgcn_s_waitcnt(0x3f70);  // vmcnt(0): q and the pages are here
  issue(pages, 0, it.begin, 0);
  int buf = 0, at = 0;  // at: the tile's first block in its batch
  for (int key0 = it.begin; key0 < it.end; key0 += KT, buf ^= 1) {
    __builtin_amdgcn_s_waitcnt(0x3f70);  // vmcnt(0): this wave's part of the tile, and the next pages
    __syncthreads();                     // everybody's, and the other tile is read
    const bool last = at == 64 - NB;     // of the batch
    if (key0 + KT < it.end) issue(last ? next : pages, last ? 0 : at + NB, key0 + KT, buf ^ 1);
    if (at == 64 - 2 * NB) next = batch(key0 + 2 * KT);
    int page[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) page[b] = page_at(pages, at + b);
    if (last) pages = next;
    at = last ? 0 : at + NB;
    const char *kt = lds + buf * 2 * TILE, *vt = kt + TILE;
    // Operands are read a phase ahead of the products that take them, which the barriers
    // below keep in place: read where they are needed, LDS's latency would be waited for
    // again and again with two waves to a SIMD.
    uint4 kk[NB][NC];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c) kk[b][c] = *reinterpret_cast<const uint4*>(kt + b * 16 * HDP * 2 + (kread ^ (c << 6)));
    __builtin_amdgcn_sched_barrier(0);
    // each sum's next product comes as late as possible: one waits for the other's result
    __builtin_amdgcn_s_setprio(1);
    f32x4_t s[NB][NT];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      // a block that is not seen (its keys read as zeros): -inf
      const float none = page[b] < 0 ? -INFINITY : 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) s[b][t] = f32x4_t{none, none, none, none};
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) s[b][t] = mfma32<C>(kk[b][c], qf[t][c], s[b][t]);
    uint4 vv[NO];
    auto read_v = [&](int b) {
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        typedef __attribute__((address_space(3))) s16x4_t* lds_t;
        const char* p = vt + b * 16 * HDP * 2 + (vread ^ (i << 5));
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p)));
        const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + 16 * HDP * 2)));
        vv[i] = make_uint4(x.x, x.y, y.x, y.y);
      }
    };
    read_v(0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[b][t][r]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = halves_max(top);
      // the reference moves where it has fallen behind by more than 2^LAG alone: weights up to
      // that are as exact, and most tiles raise some row's maximum by a little
      if (__any(top * scale > ms[t] + (LIFT + LAG) || st.m[t] == -INFINITY)) {
        const float mn = fmaxf(st.m[t], top), mns = mn == -INFINITY ? -LIFT : fmaf(mn, scale, -LIFT);
        const float alpha = st.m[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[t] - mns);
        st.m[t] = mn;
        ms[t] = mns;
        st.l[t] *= alpha;
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) st.o[t][i][r] *= alpha;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[b][t][r] = __builtin_amdgcn_exp2f(fmaf(s[b][t][r], scale, -ms[t]));
          st.l[t] += s[b][t][r];
        }
    }
#pragma unroll
    for (int b = 0; b < NB; b += 2) {
      uint4 hi[NT], lo[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) two_terms<C>(s[b][t], s[b + 1][t], hi[t], lo[t]);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) st.o[t][i] = mfma32<C>(vv[i], hi[t], st.o[t][i]);
#pragma unroll
      for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) st.o[t][i] = mfma32<C>(vv[i], lo[t], st.o[t][i]);
      __builtin_amdgcn_s_setprio(0);
      if (b + 2 < NB) {
        read_v(b + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    st.l[t] += __shfl_xor(st.l[t], 16);
    st.l[t] = halves_sum(st.l[t]);
    if (st.m[t] != -INFINITY) st.m[t] = ms[t];
  }
  __syncthreads();  // the LDS is free
}

__device__ __host__ __forceinline__ int row4(int hd) { return (hd + 3) & ~3; }
// Rows of a B slot: an even number, so that its outputs begin at 16 bytes.
__device__ __host__ __forceinline__ int cap_b(int G) { return G < 16 ? (G + 1) & ~1 : 16; }

// A slot of `cap` rows: maxima, sums, outputs.
template <int HDP, int NT, int RW>
__device__ __forceinline__ void write_slot(const PrefixArgs& a, const Item& it, const State<HDP, NT>& st, float* slot, int cap) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g4 = lane >> 4;
  if (RW == 1 && wave > 0) return;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (RW == 1 ? 0 : wave * 16 * NT) + 16 * t + col;
    if (r >= it.rows) continue;
    if (g4 == 0) {
      slot[r] = st.m[t];
      slot[cap + r] = st.l[t];
    }
#pragma unroll
    for (int i = 0; i < HDP / 16; ++i) {
      const int d = 16 * i + 4 * g4;
      if (d < row4(a.hd)) *reinterpret_cast<f32x4_t*>(slot + 2 * cap + r * row4(a.hd) + d) = st.o[t][i];
    }
  }
}

template <typename C>
__device__ __forceinline__ C* out_row(const PrefixArgs& a, int n, int head) {
  return reinterpret_cast<C*>(a.out + n * a.o_st[0] + static_cast<int64_t>(head) * a.o_st[1]);
}

// A whole B item, normalised; a request without keys gets zeros.
template <typename C, int HDP>
__device__ __forceinline__ void write_out(const PrefixArgs& a, const Item& it, const State<HDP, 1>& st) {
  const int lane = threadIdx.x & 63, col = lane & 15, g4 = lane >> 4;
  if (threadIdx.x >= 64 || col >= it.rows) return;
  C* out = out_row<C>(a, it.n0, it.h * a.G + it.row0 + col);
#pragma unroll
  for (int i = 0; i < HDP / 16; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * i + 4 * g4 + r;
      if (d < a.hd) out[d] = from_f32<C>(st.l[0] == 0.f ? 0.f : st.o[0][i][r] / st.l[0]);
    }
}

__device__ __forceinline__ int rounds_of(int keys) { return keys / kRound + (keys % kRound != 0); }

// How B's rounds are dealt out: `beside` to each workgroup that has pieces of A, `per` to
// the others.
struct Deal {
  int wgs_a, beside, per;
  __device__ __forceinline__ int64_t first(int w) const {
    return static_cast<int64_t>(min(w, wgs_a)) * beside + static_cast<int64_t>(max(w - wgs_a, 0)) * per;
  }
  __device__ __forceinline__ int of(int u) const {
    const int64_t a = static_cast<int64_t>(wgs_a) * beside;
    return u < a ? u / beside : wgs_a + (u - static_cast<int>(a)) / per;
  }
};

// The workgroups that worked on an item of r rounds that begins at u.
struct Parts {
  int first, count;
  bool inside;  // the first one begins inside its workgroup's range
};
__device__ __forceinline__ Parts parts_of(int u, int r, const Deal& d) {
  Parts p{d.of(u), 0, false};
  p.count = r == 0 ? 0 : d.of(u + r - 1) - p.first + 1;
  p.inside = u != d.first(p.first);
  return p;
}

// Whether A items of many rows go through item_rows.
template <typename C, typename KV>
constexpr bool by_rows(bool vec) { return std::is_same<C, KV>::value && sizeof(C) == 2 && vec; }

template <typename C, typename KV, int HDP>
constexpr int lds_bytes(int nt, int rw, bool vec, int nw = 4) {
  const bool f32 = sizeof(C) == 4;
  const int tile = tile_keys(HDP, f32) * pitch_of(HDP, f32) * (f32 ? 4 : 2);
  if (rw == 4 && by_rows<C, KV>(vec)) return 4 * rows_tile(HDP) * HDP * 2;
  return rw == 1 ? std::max(nw * tile, nw / 2 * 64 * nt * (2 + HDP / 4) * 4) : 2 * tile;
}

// One workgroup per B item, no split.  Few items get as many waves as registers and LDS
// let one have: 4/1 heads of 64 by 1024 keys 10.2 us with 16 waves, 12.5 with 4; where
// items fill the CUs 4 waves waste less (48 requests of 8 key heads of 128 by 512 keys:
// 18.3 us, with 8 waves 22.3).
constexpr int whole_waves(int hdp) { return hdp <= 64 ? 16 : hdp == 128 ? 8 : 4; }

template <typename C, typename KV, int HDP, bool VEC, int NW>
__global__ __launch_bounds__(64 * NW) void prefix_whole_kernel(PrefixArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[lds_bytes<C, KV, HDP>(1, 1, VEC, NW)];
  const int item = a.first + blockIdx.x, gb = item % a.GB, h = item / a.GB % a.Hkv, n = item / a.GB / a.Hkv;
  Item it{n, h, 16 * gb, min(16, a.G - 16 * gb), n, 0, clamp_len(a, a.lengths[n])};
  State<HDP, 1> st;
  item_keys<C, KV, HDP, 1, 1, VEC, NW>(a, it, lds, st);
  write_out<C, HDP>(a, it, st);
}

// Waves of a SIMD that registers are to suffice for.  256 channels without groups: 70.5 us
// with 1, 81 with 2 (60 dwords spilt; 64 requests of 8192 keys, 4/1 heads in e4m3, pages out
// of the caches).  64 channels come to 3 by themselves: 68.8 us (64 x 16384 keys), with 4 the same.
// With groups 2 is not reached where two workgroups do not fit in a CU's LDS: 16-bit queries
// with 256 channels and fp32 ones with 128 take 81980 bytes each, the plan's arrays among them.
// What is spilt: fp32 queries with 256 channels and groups 121 and 161 registers over fp32, 9
// and 16 over 8 bits; in the element-by-element forms of 256 channels with groups 262 to 364 in
// fp32 and 6 to 57 in 16 bits, 72 and 74 in 16 bits over 8 without groups; at most 5 elsewhere.
constexpr int split_waves(int hdp, int rw) { return rw == 0 && hdp == 256 ? 1 : 2; }

// Split form; RW 0: without groups.
template <typename C, typename KV, int HDP, int RW, bool VEC>
__global__ __launch_bounds__(kThreads, split_waves(HDP, RW)) void prefix_split_kernel(PrefixArgs a) {
  constexpr int NT = tiles_a(HDP, sizeof(C) == 4), RA = RW == 0 ? 1 : RW, ROWS = 16 * NT * RA;
  constexpr int LDS_A = RW == 0 ? 0 : lds_bytes<C, KV, HDP>(NT, RA, VEC), LDS_B = lds_bytes<C, KV, HDP>(1, 1, VEC);
  __shared__ __attribute__((aligned(16))) char lds[LDS_A > LDS_B ? LDS_A : LDS_B];
  // prefix sums of the groups' rounds and pieces, and of the requests' own rounds
  __shared__ int units[RW == 0 ? 1 : kRequests + 1], pre_b[kRequests + 1];
  // the first request of a group that has the whole prefix, and the keys read once (0: nobody has it)
  __shared__ uint16_t lead[RW == 0 ? 1 : kRequests];
  __shared__ int keys[RW == 0 ? 1 : kRequests];
  __shared__ Deal s_deal;
  __shared__ int wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto scan = [&](int n, int* pre, auto&& value) {  // pre[i + 1] = value(0) + .. + value(i)
    int base = 0;
    if (tid == 0) pre[0] = 0;
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const int i = i0 + tid;
      int s = wave_incl_sum(i < n ? value(i) : 0);
      if (lane == 63) wsum[wave] = s;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < 4; ++w) {
        if (w < wave) s += wsum[w];
        all += wsum[w];
      }
      if (i < n) pre[i + 1] = base + s;
      base += all;
      __syncthreads();
    }
  };
  const int HA = a.Hkv * a.RB, HB = a.Hkv * a.GB;
  // the last x with pre[x] <= u
  auto find = [](const int* pre, int n, int u) {
    int x = 0;
    for (int hi = n; hi - x > 1;) {
      const int mid = (x + hi) >> 1;
      if (pre[mid] <= u) x = mid; else hi = mid;
    }
    return x;
  };
  auto own_begin = [&](int n) {  // where request n's own keys begin
    if constexpr (RW == 0) return 0;
    const int g = n / a.W;
    return clamp_len(a, a.lengths[n]) >= clamp_len(a, a.shared[g]) ? shared_keys(a, g) : 0;
  };
  // How long the pieces are, and how B is dealt out; next_units(per) makes `units` for
  // pieces of up to `per` rounds and returns their number.  (All of these counts stay below
  // 2^31, which the host sees to: a 64-bit division here and there took longer than the keys.)
  auto deal_out = [&](int rounds_a, int total_b, auto&& next_units) {
    Deal d{0, 0, 1};
    if (rounds_a > 0) {
      // The least piece for which the pieces are no more than the workgroups, so that each
      // has one, if all items are not more than that already.
      const unsigned all_rounds = rounds_a * HA;
      const bool fit = a.groups * HA <= a.wgs;
      int per = (all_rounds + a.wgs - 1) / a.wgs, all = 0;
      for (int turn = 0; turn < 16; ++turn) {
        all = next_units(per) * HA;
        if (all <= a.wgs || !fit) break;
        per = max(per + 1, static_cast<int>(static_cast<float>(per) * static_cast<float>(all) / static_cast<float>(a.wgs)));
      }
      d.wgs_a = min(a.wgs, all);
      // B rounds that take a workgroup as long as its pieces: a round of A is RW tiles
      // of a wave, one of B a single one
      const int busy = all_rounds * RW / d.wgs_a, rest = a.wgs - d.wgs_a;
      const int64_t filled = static_cast<int64_t>(busy) * rest;
      if (total_b <= filled) {
        d.per = rest == 0 ? 1 : (total_b + rest - 1) / rest;
      } else {
        d.beside = (total_b - static_cast<int>(filled) + a.wgs - 1) / a.wgs;
        d.per = busy + d.beside;
      }
    } else {
      d.per = (total_b + a.wgs - 1) / a.wgs;
    }
    d.per = max(d.per, 1);
    return d;
  };
  if (a.N <= 64) {  // in the lanes of one wave
    if (wave == 0) {
      const int len = lane < a.N ? clamp_len(a, a.lengths[lane]) : 0;
      int begin = 0, rounds_a = 0, rounds = 0;
      if constexpr (RW != 0) {
        const int own = lane < a.N ? clamp_len(a, a.shared[lane / a.W]) : 0, mine = lane < a.groups ? clamp_len(a, a.shared[lane]) : 0;
        const bool has = lane < a.N && len >= own;
        begin = has ? own & ~15 : 0;
        const uint64_t who = __ballot(has);
        const uint64_t of_group = lane < a.groups ? who >> (lane * a.W) & (~0ull >> (64 - a.W)) : 0;
        const int first = of_group ? lane * a.W + __ffsll(static_cast<unsigned long long>(of_group)) - 1 : a.N;
        const int seen = of_group ? mine & ~15 : 0;
        if (lane < a.groups) {
          lead[lane] = static_cast<uint16_t>(first);
          keys[lane] = seen;
        }
        rounds = rounds_of(seen);
        rounds_a = __builtin_amdgcn_readlane(wave_incl_sum(rounds), 63);
      }
      const int upto = wave_incl_sum(lane < a.N ? rounds_of(len - begin) : 0);
      if (lane < a.N) pre_b[lane + 1] = upto;
      if (lane == 0) pre_b[0] = 0;
      const Deal d = deal_out(rounds_a, __builtin_amdgcn_readlane(upto, 63) * HB, [&](int per) {
        const int s = wave_incl_sum((rounds + per - 1) / per);
        if (RW != 0 && lane < a.groups) units[lane + 1] = s;
        return static_cast<int>(__builtin_amdgcn_readlane(s, 63));
      });
      if (lane == 0) {
        s_deal = d;
        if constexpr (RW != 0) units[0] = 0;
      }
      if (RW != 0 && rounds_a == 0 && lane < a.groups) units[lane + 1] = 0;
    }
    __syncthreads();
  } else {
    int rounds_a = 0;
    if constexpr (RW != 0) {
      for (int g = tid; g < a.groups; g += kThreads) keys[g] = a.N;
      __syncthreads();
      for (int n = tid; n < a.N; n += kThreads) {
        const int g = n / a.W;
        if (clamp_len(a, a.lengths[n]) >= clamp_len(a, a.shared[g])) atomicMin(&keys[g], n);
      }
      __syncthreads();
      for (int g = tid; g < a.groups; g += kThreads) {
        const int first = keys[g];
        lead[g] = static_cast<uint16_t>(first);
        keys[g] = first < a.N ? shared_keys(a, g) : 0;
      }
      __syncthreads();
      scan(a.groups, units, [&](int g) { return rounds_of(keys[g]); });
      rounds_a = units[a.groups];
      __syncthreads();  // read before it is written again
    }
    scan(a.N, pre_b, [&](int n) { return rounds_of(clamp_len(a, a.lengths[n]) - own_begin(n)); });
    const Deal d = deal_out(rounds_a, pre_b[a.N] * HB, [&](int per) {
      scan(a.groups, units, [&](int g) { return (rounds_of(keys[g]) + per - 1) / per; });
      const int all = units[a.groups];
      __syncthreads();
      return all;
    });
    if (tid == 0) s_deal = d;
    __syncthreads();
  }
  const Deal deal = s_deal;
  const int total_b = pre_b[a.N] * HB, units_a = RW == 0 ? 0 : units[a.groups] * HA;
  if (blockIdx.x == 0) {  // for the joining kernel
    if (tid == 0) {
      a.plan[kWgsA] = deal.wgs_a;
      a.plan[kBeside] = deal.beside;
      a.plan[kPer] = deal.per;
    }
    if constexpr (RW != 0)
      for (int i = tid; i <= a.groups; i += kThreads) a.plan[kPlan + i] = units[i];
    for (int i = tid; i <= a.N; i += kThreads) a.plan[kPlan + a.groups + 1 + i] = pre_b[i];
  }
  if constexpr (RW != 0) {
    const int wgs_a = deal.wgs_a;
    if (static_cast<int>(blockIdx.x) < wgs_a) {
      // Pieces in the order (group, key head, piece, block of rows), each XCD (workgroups go
      // to them in turn) a run of them: the blocks of rows read the same keys from its L2.
      const int w = blockIdx.x, xcds = min(8, wgs_a), x = w % xcds, at = w / xcds, beside = (wgs_a - x + xcds - 1) / xcds;
      const int some = units_a / xcds, more = units_a - some * xcds;
      const int first = some * x + min(x, more), last = some * (x + 1) + min(x + 1, more);
      for (int u = first + at; u < last; u += beside) {
        const int g = find(units, a.groups, u / HA);
        const int pieces = units[g + 1] - units[g], r = rounds_of(keys[g]), v = u - units[g] * HA;
        const int h = v / (pieces * a.RB), y = v - h * pieces * a.RB, piece = y / a.RB, rb = y - piece * a.RB;
        const int each = r / pieces, over = r - each * pieces;
        const int t0 = each * piece + min(piece, over), t1 = each * (piece + 1) + min(piece + 1, over);
        Item it{g * a.W, h, rb * ROWS, min(ROWS, a.W * a.G - rb * ROWS), lead[g], t0 * kRound,
                t1 == r ? keys[g] : t1 * kRound};
        State<HDP, NT> st;
        if constexpr (RW == 4 && by_rows<C, KV>(VEC)) item_rows<C, HDP, NT>(a, it, lds, st);
        else item_keys<C, KV, HDP, NT, RA, VEC>(a, it, lds, st);
        write_slot<HDP, NT, RA>(a, it, st, a.part + u * a.slot_a, ROWS);
      }
    }
  }
  const int begin = min(deal.first(blockIdx.x), static_cast<int64_t>(total_b));
  const int end = min(deal.first(blockIdx.x + 1), static_cast<int64_t>(total_b));
  int n = begin < end ? find(pre_b, a.N, begin / HB) : 0;
  for (int u = begin; u < end;) {
    while (pre_b[n + 1] * HB <= u) ++n;
    const int r = pre_b[n + 1] - pre_b[n], at = u - pre_b[n] * HB, hg = at / r, t0 = at - hg * r;
    const int take = min(r - t0, end - u);
    const bool all = take == r;
    const int h = hg / a.GB, gb = hg - h * a.GB, len = clamp_len(a, a.lengths[n]), own = own_begin(n);
    // a long context's last round may end past an int
    const int last = len - own - t0 * kRound > take * kRound ? own + (t0 + take) * kRound : len;
    Item it{n, h, 16 * gb, min(16, a.G - 16 * gb), n, own + t0 * kRound, last};
    State<HDP, 1> st;
    item_keys<C, KV, HDP, 1, 1, VEC>(a, it, lds, st);
    if (RW == 0 && all) {
      write_out<C, HDP>(a, it, st);
    } else {
      float* to = a.part + (all ? a.whole_b + (static_cast<int64_t>(n) * HB + hg) * a.slot_b
                                : a.part_b + (static_cast<int64_t>(blockIdx.x) * 2 + (u == begin ? 0 : 1)) * a.slot_b);
      write_slot<HDP, 1, 1>(a, it, st, to, cap_b(a.G));
    }
    u += take;
  }
}

// Joins a row's parts, the prefix's first, each in its order; TPR threads a row,
// four elements each, the parts dealt out over the threads left.  Zeros where no
// key was seen.  Without groups, items that one workgroup had whole are written.
template <typename C, int TPR>
__global__ __launch_bounds__(kThreads) void prefix_join_kernel(PrefixArgs a, int rows_a) {
  constexpr int ROWS = kThreads / TPR, WAVES = TPR / 64;
  __shared__ float4 sums[TPR > 64 ? TPR : 1];
  __shared__ float lsum[TPR > 64 ? TPR : 1], tops[WAVES];
  const int tid = threadIdx.x % TPR, lane = threadIdx.x & 63, wave = tid >> 6;
  const int row = blockIdx.x * ROWS + threadIdx.x / TPR;
  if (row >= a.N * a.H) return;  // whole waves; where threads meet, ROWS is 1
  const int n = row / a.H, head = row - n * a.H, h = head / a.G, g = head - h * a.G;
  const int HA = a.Hkv * a.RB, HB = a.Hkv * a.GB;
  const Deal deal{a.plan[kWgsA], a.plan[kBeside], a.plan[kPer]};
  int pieces = 0, at_a = 0;
  const float* part_a = nullptr;
  if (a.groups != 0) {
    const int x = n / a.W, u0 = a.plan[kPlan + x];
    if (clamp_len(a, a.lengths[n]) >= clamp_len(a, a.shared[x])) {
      const int m = (n - x * a.W) * a.G + g, rb = m / rows_a;
      at_a = m - rb * rows_a;
      pieces = a.plan[kPlan + x + 1] - u0;
      part_a = a.part + (static_cast<int64_t>(u0) * HA + static_cast<int64_t>(h) * pieces * a.RB + rb) * a.slot_a;
    }
  }
  const int* pre_b = a.plan + kPlan + a.groups + 1;
  const int gb = g >> 4, at_b = g & 15, hg = h * a.GB + gb, r = pre_b[n + 1] - pre_b[n];
  const Parts pb = parts_of(pre_b[n] * HB + hg * r, r, deal);
  if (a.groups == 0 && pb.count == 1) return;
  const float* whole_b = pb.count == 1 ? a.part + a.whole_b + (static_cast<int64_t>(n) * HB + hg) * a.slot_b : nullptr;
  const int parts = pieces + pb.count, r4 = row4(a.hd);
  struct At { const float *m, *l, *o; };
  auto part = [&](int p) {
    const bool is_a = p < pieces;
    const int i = p - pieces;
    const float* s = is_a ? part_a + static_cast<int64_t>(p) * a.RB * a.slot_a
                     : whole_b ? whole_b
                               : a.part + a.part_b +
                                     (static_cast<int64_t>(pb.first + i) * 2 + (i == 0 && pb.inside ? 1 : 0)) * a.slot_b;
    const int cap = is_a ? rows_a : cap_b(a.G), at = is_a ? at_a : at_b;
    return At{s + at, s + cap + at, s + 2 * cap + at * r4};
  };
  float top = -INFINITY;
  for (int p = tid; p < parts; p += TPR) top = fmaxf(top, *part(p).m);
  top = wave_max(top);
  if constexpr (TPR > 64) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
  }
  const float ts = top == -INFINITY ? 0.f : top;
  const int quads = r4 / 4;
  int qp = 1;
  while (qp < quads) qp *= 2;
  const int e = tid & (qp - 1), sub = tid / qp, subs = TPR / qp;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (e < quads) {
#pragma unroll 4
    for (int p = sub; p < parts; p += subs) {
      const At s = part(p);
      const float c = __builtin_amdgcn_exp2f(*s.m - ts);
      const float4 x = *reinterpret_cast<const float4*>(s.o + 4 * e);
      l = fmaf(c, *s.l, l);
      o.x = fmaf(c, x.x, o.x);
      o.y = fmaf(c, x.y, o.y);
      o.z = fmaf(c, x.z, o.z);
      o.w = fmaf(c, x.w, o.w);
    }
  }
  for (int off = qp; off < 64; off *= 2) {
    o.x += __shfl_xor(o.x, off);
    o.y += __shfl_xor(o.y, off);
    o.z += __shfl_xor(o.z, off);
    o.w += __shfl_xor(o.w, off);
    l += __shfl_xor(l, off);
  }
  if constexpr (TPR > 64) {
    sums[tid] = o;
    lsum[tid] = l;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < WAVES; ++w) {
        const float4 x = sums[64 * w + lane];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
        l += lsum[64 * w + lane];
      }
    }
  }
  if (wave == 0 && lane < quads) {
    C* out = out_row<C>(a, n, head) + 4 * lane;
    const float v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * lane + i < a.hd) out[i] = from_f32<C>(l == 0.f ? 0.f : v[i] / l);
  }
}

// ------------------------------------------------------------------- launch
struct Shape {
  int hdp, rw, rows_a;  // rw: 0 without groups
  bool vec;
};

// Rows that 16-byte loads cannot take come element by element, in forms of 64 and 256
// channels.
inline Shape shape_of(int64_t hd, int64_t G, int64_t W, bool groups, int e, bool vec) {
  Shape s{};
  s.vec = vec;
  s.hdp = !vec ? (hd <= 64 ? 64 : 256) : hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
  const int nt = tiles_a(s.hdp, e == 4);
  // 16 bits of the queries' own type: as fast either way (8 groups of 16 rows by 1500 keys of 64: 12.6 us);
  // 8 bits 13.0 : 15.6 there, fp32 15.0 : 21.7
  s.rw = !groups ? 0 : W * G <= 16 * nt ? 1 : 4;
  s.rows_a = 16 * nt * (s.rw == 4 ? 4 : 1);
  return s;
}

template <typename C, typename KV, int HDP, int RW, bool VEC>
int launch_split(PrefixArgs a, int rows_a, hipStream_t st) {
  const auto kernel = prefix_split_kernel<C, KV, HDP, RW, VEC>;
  a.wgs = std::min(a.wgs, a.cus * blocks_per_cu(reinterpret_cast<const void*>(kernel), kThreads));
  kernel<<<a.wgs, kThreads, 0, st>>>(a);
  const int64_t rows = static_cast<int64_t>(a.N) * a.H;
  // a workgroup or a wave to a row: 8 rows of 32768 keys 13.6 : 23.0 us (with the split), 256 rows of 8192
  // 25.7 : 26.8, 384 rows 29.1 : 28.8, 8000 rows 480 : 473
  if (rows <= 256) prefix_join_kernel<C, 256><<<static_cast<unsigned>(rows), 256, 0, st>>>(a, rows_a);
  else prefix_join_kernel<C, 64><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, st>>>(a, rows_a);
  return check_launch("prefix_attn");
}

template <typename C, typename KV, int HDP, bool VEC>
int launch_form(const PrefixArgs& a, const Shape& s, hipStream_t st) {
  if (s.rw == 1) return launch_split<C, KV, HDP, 1, VEC>(a, s.rows_a, st);
  if (s.rw == 4) return launch_split<C, KV, HDP, 4, VEC>(a, s.rows_a, st);
  if constexpr (sizeof(KV) == 1) {
    if (a.split) return launch_split<C, KV, HDP, 0, VEC>(a, s.rows_a, st);
    PrefixArgs b = a;
    const int64_t items = static_cast<int64_t>(a.N) * a.Hkv * a.GB;
    constexpr int64_t most = int64_t(1) << 22;  // HIP counts a launch's threads in 32 bits
    for (int64_t first = 0; first < items; first += most) {
      b.first = static_cast<int>(first);
      const unsigned wgs = static_cast<unsigned>(std::min(most, items - first));
      if (a.waves == 4) prefix_whole_kernel<C, KV, HDP, VEC, 4><<<wgs, kThreads, 0, st>>>(b);
      else prefix_whole_kernel<C, KV, HDP, VEC, whole_waves(HDP)><<<wgs, 64 * whole_waves(HDP), 0, st>>>(b);
    }
    return check_launch("prefix_attn");
  }
  return fail(HYDRA_ERR_ARG, "prefix_attn: pages of the queries' type without groups");
}

template <typename C, typename KV>
int launch_pages(const PrefixArgs& a, const Shape& s, hipStream_t st) {
  if (!s.vec && s.hdp == 64) return launch_form<C, KV, 64, false>(a, s, st);
  if (!s.vec) return launch_form<C, KV, 256, false>(a, s, st);
  switch (s.hdp) {
    case 32: return launch_form<C, KV, 32, true>(a, s, st);
    case 64: return launch_form<C, KV, 64, true>(a, s, st);
    case 128: return launch_form<C, KV, 128, true>(a, s, st);
    default: return launch_form<C, KV, 256, true>(a, s, st);
  }
}

// One file each instantiates it for a type of the queries and of the pages.
#define HYDRA_PREFIX_TYPES(X)                                                                                    \
  X(float, float) X(float, i8) X(float, e4m3) X(bf16, bf16) X(bf16, i8) X(bf16, e4m3) X(f16, f16) X(f16, i8) X(f16, e4m3)
#define HYDRA_PREFIX_EXTERN(C, KV) extern template int launch_pages<C, KV>(const PrefixArgs&, const Shape&, hipStream_t);
HYDRA_PREFIX_TYPES(HYDRA_PREFIX_EXTERN)

}  // namespace prefix
}  // namespace hydra
