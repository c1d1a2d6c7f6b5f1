// One token of CCGQA attention's q/k/v preparation on gfx950, for requests that
// are decoded: what ccgqa_prep.hip does for whole sequences
// (hydra/attention/backends/ccgqa/attention.py:205-266, kernels/fused_conv.py:39-62),
// for the newest token of each request, with the rows before it taken from a
// ring and k and v written to the request's slot in a paged cache.
//
// With x_d the projected row d tokens back (zero before the sequence began),
//   y1[j] = sum_t W1[t] x[2(ks-1) - j - t]   (grouped by head), j = 0 .. ks-1
//   y2    = sum_j W2[j] y1[j]                (dense)
//   q, k  = rope(normalize(y2 + QK-mean) (* temperature)), v = v_curr | v_prev.
// y1 is computed again at its ks positions: that is ks^2 hd products a channel
// beside the ks C of conv2, and leaves one launch and a state of plain rows.
// fp32 throughout, one rounding at the end, but that the matrix form of a 16-bit
// type carries y1 into conv2 as two terms of it: 16 significant bits for bf16; for
// fp16 22 from 1/8 on, to within 2^-25 below, and infinity beyond fp16's range.
// The prompts' kernels keep one such term.
//
// The ring holds each request's last R projected rows, row p at p % R.  A step
// reads rows p - 2(ks-1) .. p-1 and writes row p, which is none of them as R >
// 2(ks-1): the workgroups of a launch need no order.
#include "common.h"

#include <algorithm>

namespace hydra {
namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

struct DecodeArgs {
  const void* qkv;
  int64_t qkv_rs;
  void* ring;  // [N, R, W]
  const int* positions;
  const int64_t* slots;
  const void *w[4];  // wq1, wq2, wk1, wk2, tap-major or tiled
  const void *temp, *cos, *sin;
  int64_t cs_rs;
  void *q, *kp, *vp;
  int64_t kps[3], vps[3];  // elements: page, h, row
  int64_t limit;           // slots of the pool
  int N, R, Hq, Hkv, hd, ks, shift, rope_rows, flags;
  int span;     // matrix-core form: channel blocks of a workgroup
  float* part;  // sums of heads that several workgroups share
};

// The token that request n's newest row stands at, or -1: no slot of the pool,
// or a position that the rotation's table does not hold.
__device__ __forceinline__ int active_position(const DecodeArgs& a, int n) {
  if (n >= a.N) return -1;
  const int p = a.positions[n];
  const int64_t slot = a.slots[n];
  const bool ok = p >= 0 && slot >= 0 && slot < a.limit && (!(a.flags & HYDRA_CCGQA_ROPE) || p < a.rope_rows);
  return ok ? p : -1;
}

// Row `back` tokens before position p of request n (the caller checks back <= p).
template <typename T>
__device__ __forceinline__ const T* row_at(const DecodeArgs& a, int n, int p, int back) {
  if (back == 0) return static_cast<const T*>(a.qkv) + n * a.qkv_rs;
  const int W = (a.Hq + 2 * a.Hkv) * a.hd;
  return static_cast<const T*>(a.ring) + (static_cast<int64_t>(n) * a.R + (p - back) % a.R) * W;
}

// QK-mean's term of channel d of head `hh` (k heads from Hq on) from the newest row.
template <typename T>
__device__ __forceinline__ float mean_term(const DecodeArgs& a, const T* row, int hh, int d) {
  const int L = a.Hq * a.hd;
  if (a.Hq == a.Hkv) {
    const int h = hh < a.Hq ? hh : hh - a.Hq;
    return 0.5f * (to_f32(row[h * a.hd + d]) + to_f32(row[L + h * a.hd + d]));
  }
  const bool is_k = hh >= a.Hq;  // q heads get the mean of k, k heads that of q
  const T* from = row + (is_k ? 0 : L) + d;
  const int heads = is_k ? a.Hq : a.Hkv;
  float s = 0.f;
  for (int h = 0; h < heads; ++h) s += to_f32(from[h * a.hd]);
  return 0.5f * s / static_cast<float>(heads);
}

__device__ __forceinline__ void rope_at(const DecodeArgs& a, int p, int i, float& c, float& s) {
  const int64_t at = static_cast<int64_t>(p) * a.cs_rs + i;
  if (a.flags & HYDRA_CCGQA_ROPE_BF16) {
    c = to_f32(static_cast<const bf16*>(a.cos)[at]);
    s = to_f32(static_cast<const bf16*>(a.sin)[at]);
  } else {
    c = static_cast<const float*>(a.cos)[at];
    s = static_cast<const float*>(a.sin)[at];
  }
}

// Channel c of v.
template <typename T>
__device__ __forceinline__ T value_at(const DecodeArgs& a, int n, int p, int c) {
  const int K = a.Hkv * a.hd, at = a.Hq * a.hd + K;
  const T* row = row_at<T>(a, n, p, 0);
  if (!(a.flags & HYDRA_CCGQA_VALUE_SHIFT) || c < K / 2) return row[at + c];
  return p > 0 ? row_at<T>(a, n, p, 1)[at + c] : from_f32<T>(0.f);
}

// Everything after the convs, for one request and head, by one wave (lane i
// has the channel pairs i, i + 64, ...); y(d) gives conv2's channel d.
template <typename T, typename Y>
__device__ __forceinline__ void finish(const DecodeArgs& a, int n, int p, int hh, int lane, Y y) {
  const bool is_k = hh >= a.Hq;
  const int head = is_k ? hh - a.Hq : hh, pairs = a.hd / 2;
  T* qrow = is_k ? nullptr : static_cast<T*>(a.q) + (static_cast<int64_t>(n) * a.Hq + head) * a.hd;
  if (p < 0) {
    if (!is_k)
      for (int d = lane; d < a.hd; d += 64) qrow[d] = from_f32<T>(0.f);
    return;
  }
  const T* row = row_at<T>(a, n, p, 0);
  const bool mean = a.flags & HYDRA_CCGQA_QK_MEAN;
  float gain = 1.f;
  if (a.flags & HYDRA_CCGQA_QK_NORM) {
    float s = 0.f;
    for (int i = lane; i < pairs; i += 64)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float v = y(2 * i + e) + (mean ? mean_term<T>(a, row, hh, 2 * i + e) : 0.f);
        s = fmaf(v, v, s);
      }
    s = wave_sum(s);
    gain = 1.f / fmaxf(sqrtf(s), 1e-12f);  // F.normalize's eps
    if (is_k) gain *= to_f32(*static_cast<const T*>(a.temp));
  }
  T *out = qrow, *vout = nullptr;
  if (is_k) {
    const int64_t slot = a.slots[n], page = slot >> a.shift, r = slot & ((int64_t(1) << a.shift) - 1);
    out = static_cast<T*>(a.kp) + page * a.kps[0] + head * a.kps[1] + r * a.kps[2];
    vout = static_cast<T*>(a.vp) + page * a.vps[0] + head * a.vps[1] + r * a.vps[2];
  }
  for (int i = lane; i < pairs; i += 64) {
    float v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      v[e] = (y(2 * i + e) + (mean ? mean_term<T>(a, row, hh, 2 * i + e) : 0.f)) * gain;
    if (a.flags & HYDRA_CCGQA_ROPE) {
      float c, s;
      rope_at(a, p, i, c, s);
      const float x0 = v[0], x1 = v[1];
      v[0] = x0 * c - x1 * s;
      v[1] = x0 * s + x1 * c;
    }
    out[2 * i] = from_f32<T>(v[0]);
    out[2 * i + 1] = from_f32<T>(v[1]);
  }
  if (is_k)
    for (int d = lane; d < a.hd; d += 64) vout[d] = value_at<T>(a, n, p, head * a.hd + d);
}

template <typename T>
__device__ __forceinline__ void keep_row(const DecodeArgs& a, int n, int p, int tid, int threads) {
  if (p < 0) return;
  const int W = (a.Hq + 2 * a.Hkv) * a.hd;
  const T* from = row_at<T>(a, n, p, 0);
  T* to = static_cast<T*>(a.ring) + (static_cast<int64_t>(n) * a.R + p % a.R) * W;
  for (int c = tid; c < W; c += threads) to[c] = from[c];
}

// The same with 16-byte pieces (rows of whole ones, aligned), by one wave.
__device__ __forceinline__ void keep_row16(const DecodeArgs& a, int n, int p, int lane, int size) {
  if (p < 0) return;
  const int64_t bytes = static_cast<int64_t>((a.Hq + 2 * a.Hkv) * a.hd) * size;
  const uint4* from = reinterpret_cast<const uint4*>(static_cast<const char*>(a.qkv) + n * a.qkv_rs * size);
  uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(a.ring) + (static_cast<int64_t>(n) * a.R + p % a.R) * bytes);
#pragma unroll 4
  for (int c = lane; c < bytes / 16; c += 64) to[c] = from[c];
}

constexpr int kGenericThreads = 1024;

// s plus the product of n elements of a and b, in 16-byte pieces where VEC.
template <typename T, bool VEC>
__device__ __forceinline__ float dot(const T* a, const T* b, int n, float s) {
  if constexpr (VEC) {
    constexpr int E = Vec<T>::N;
#pragma unroll 4
    for (int i = 0; i < n; i += E) {
      float x[E], y[E];
      load16<T>(a + i, x);
      load16<T>(b + i, y);
#pragma unroll
      for (int k = 0; k < E; ++k) s = fmaf(x[k], y[k], s);
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < n; ++i) s = fmaf(to_f32(a[i]), to_f32(b[i]), s);
  }
  return s;
}

// Any head_dim, taps and flags: one workgroup per request and head on the
// VALU, y1 in LDS as [ks][C] floats, then y2 [hd].  Every workgroup computes all
// of conv1 for itself, ks^2 hd products a channel, and a lane's weights are rows
// of their own, so the cache's lines bound it: 8/2 heads of 48, three taps, 18 us
// for one request and 34 us for 32; heads of 64 with five taps, 32 requests, 156 us.
template <typename T, bool VEC>
__global__ __launch_bounds__(kGenericThreads) void decode_prep_generic_kernel(DecodeArgs a) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hh = blockIdx.x, n = blockIdx.y;
  const bool is_k = hh >= a.Hq;
  const int hd = a.hd, L = a.Hq * hd, C = is_k ? a.Hkv * hd : L, col0 = is_k ? L : 0;
  const int head = is_k ? hh - a.Hq : hh;
  const int p = active_position(a, n);
  const bool convs = a.flags & HYDRA_CCGQA_CONVS;
  float* y2 = sm + (convs ? a.ks * C : 0);
  if (p >= 0 && convs) {
    const T *w1 = static_cast<const T*>(a.w[is_k ? 2 : 0]), *w2 = static_cast<const T*>(a.w[is_k ? 3 : 1]);
    for (int i = tid; i < a.ks * C; i += kGenericThreads) {
      const int j = i / C, c = i - j * C, g0 = c / hd * hd;
      float s = 0.f;
      for (int t = 0; t < a.ks; ++t) {
        const int back = 2 * (a.ks - 1) - j - t;
        if (back > p) continue;
        s = dot<T, VEC>(w1 + (static_cast<int64_t>(t) * C + c) * hd, row_at<T>(a, n, p, back) + col0 + g0, hd, s);
      }
      sm[i] = s;
    }
    __syncthreads();
    for (int d = wave; d < hd; d += kGenericThreads / 64) {
      float s = 0.f;
      for (int j = 0; j < a.ks; ++j) {
        const T* w = w2 + (static_cast<int64_t>(j) * C + head * hd + d) * C;
        if constexpr (VEC) {
          constexpr int E = Vec<T>::N;
          for (int c = lane * E; c < C; c += 64 * E) {
            float x[E];
            load16<T>(w + c, x);
#pragma unroll
            for (int k = 0; k < E; ++k) s = fmaf(x[k], sm[j * C + c + k], s);
          }
        } else {
          for (int c = lane; c < C; c += 64) s = fmaf(to_f32(w[c]), sm[j * C + c], s);
        }
      }
      s = wave_sum(s);
      if (lane == 0) y2[d] = s;
    }
  } else if (p >= 0) {
    const T* x = row_at<T>(a, n, p, 0) + col0 + head * hd;
    for (int d = tid; d < hd; d += kGenericThreads) y2[d] = to_f32(x[d]);
  }
  __syncthreads();
  if (wave == 0) finish<T>(a, n, p, hh, lane, [&](int d) { return y2[d]; });
  if (hh == 0) keep_row<T>(a, n, p, tid, kGenericThreads);
}

// ---- matrix-core form: three taps, head_dim 16, 32, 64 or 128 ---------------
// Operands of 16 rows (or columns; lane & 15) and K input channels, of which lane
// group g = lane >> 4 holds K/4 neighbouring ones: v_mfma_f32_16x16x32 with K = 32
// for a 16-bit type, 16x16x16 where head_dim is 16, four 16x16x4 in fp32 (the i-th
// takes element i: k is a name that both operands share).  The result's lane
// holds column lane & 15, rows 4 g + i: the next product's operand of K = 16, so
// y1 goes from conv1 to conv2 in registers.
template <typename T, int K>
using Frag = typename std::conditional<sizeof(T) * K == 32, uint2, uint4>::type;

template <typename T>
__device__ __forceinline__ f32x4_t mma32(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}

template <typename T, int K>
__device__ __forceinline__ f32x4_t mma(Frag<T, K> a, Frag<T, K> b, f32x4_t c) {
  if constexpr (std::is_same<T, float>::value) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  } else if constexpr (K == 32) {
    return mma32<T>(a, b, c);
  } else if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c,
                                                     0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a), __builtin_bit_cast(f16x4_t, b), c, 0,
                                                 0, 0);
  }
}

// y1 as conv2's operand: fp32 as it is, a 16-bit type as the rounded value and
// what that leaves, the two halves of one K = 32 product whose other operand
// holds the weights twice.
template <typename T>
struct Y1 {
  uint4 f;
  __device__ __forceinline__ explicit Y1(f32x4_t y) {
    if constexpr (sizeof(T) == 4) {
      f = __builtin_bit_cast(uint4, y);
    } else {
      float rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float h = to_f32(from_f32<T>(y[i]));
        rest[i] = fabsf(h) == INFINITY ? 0.f : y[i] - h;
      }
      f = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(rest[0], rest[1]), pack2<T>(rest[2], rest[3]));
    }
  }
  __device__ __forceinline__ f32x4_t times(Frag<T, 16> w, f32x4_t c) const {
    if constexpr (sizeof(T) == 4) return mma<T, 16>(w, f, c);
    else return mma32<T>(make_uint4(w.x, w.y, w.x, w.y), f, c);
  }
};

// Operand block (tap t, output channels 16 ob .., input channels K ib ..) of a
// weight [3][O][I], or of its MFMA-tiled order [3][O/32][I/16][2][32][8]: a
// wave-uniform base and the lane's own 32-bit offset, which is the same for
// every block.
template <typename T, int K, bool TILED>
struct Weights {
  const char* base;
  int O, I;
  uint32_t lane_off;
  __device__ __forceinline__ Weights(const void* w, int o, int i) : base(static_cast<const char*>(w)), O(o), I(i) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    uint32_t at = r * I + K / 4 * g;
    if (TILED) at = K == 32 ? (g >> 1) * 512 + (g & 1) * 256 + r * 8 : (g >> 1) * 256 + r * 8 + (g & 1) * 4;
    lane_off = at * sizeof(T);
  }
  __device__ __forceinline__ Frag<T, K> operator()(int t, int ob, int ib) const {
    int64_t at = static_cast<int64_t>(t) * O * I;
    if (TILED) at += (static_cast<int64_t>(ob >> 1) * (I >> 4) + ib * (K / 16)) * 512 + (ob & 1) * 128;
    else at += static_cast<int64_t>(ob) * 16 * I + ib * K;
    return *reinterpret_cast<const Frag<T, K>*>(base + at * static_cast<int64_t>(sizeof(T)) + lane_off);
  }
};

// Most waves of a workgroup: all loads of a channel block of 16 are in flight at
// once (11 operands), so wide heads get twice the registers and half the waves.
constexpr int decode_waves(int hb, int size) { return hb * size <= 8 ? 16 : 8; }

// Channel blocks of a workgroup.  A CU draws weights from L2 at about 50 GB/s when
// few of them run, so a head whose weights (conv1's of all its channels, its own
// of conv2) are large is dealt out to workgroups of 4 waves and 4 blocks, and a
// second launch (4 us, what 200 KB take, or 100 KB of tap-major weights, whose
// operands are 32-byte pieces of rows) adds them up and ends the chain; not from
// 128 workgroups on (128 requests, 8/2 heads of 64, 80 workgroups split in 8: 14.0 +
// 4.0 us; 256, 160 of them whole: 19.3).
struct DecodePlan {
  int span, waves, splits;
};

DecodePlan decode_plan(int64_t N, int64_t Hq, int64_t Hkv, int64_t hd, int size, bool tiled) {
  const int64_t C = Hq * hd, blocks = C / 16, groups = (Hq + Hkv) * ((N + 15) / 16);
  DecodePlan p{};
  p.waves = decode_waves(static_cast<int>(hd / 16), size);
  p.span = static_cast<int>(blocks);
  if (6 * C * hd * size > (tiled ? 200 : 100) * 1024 && groups < 128) {
    p.waves = 4;
    p.span = 4;
  }
  if (p.waves > blocks) p.waves = blocks < 4 ? 4 : static_cast<int>(blocks);
  p.splits = static_cast<int>((blocks + p.span - 1) / p.span);
  return p;
}

// Two neighbouring channels.
template <typename T>
struct Pair {
  float v[2];
  __device__ __forceinline__ explicit Pair(const T* at) {
    if constexpr (sizeof(T) == 4) {
      const float2 f = *reinterpret_cast<const float2*>(at);
      v[0] = f.x;
      v[1] = f.y;
    } else {
      const uint32_t raw = *reinterpret_cast<const uint32_t*>(at);
      T lo, hi;
      lo.bits = static_cast<uint16_t>(raw & 0xffffu);
      hi.bits = static_cast<uint16_t>(raw >> 16);
      v[0] = to_f32(lo);
      v[1] = to_f32(hi);
    }
  }
};

// QK-mean's terms of a head of the requests n0 .. n0+15 to mean [HD][17], by all
// threads: heads are summed eight loads at a time.
template <typename T, int HD>
__device__ __forceinline__ void mean_fill(const DecodeArgs& a, int n0, int hh, int threads, float (*mean)[17]) {
  if (!(a.flags & HYDRA_CCGQA_QK_MEAN)) return;
  const bool is_k = hh >= a.Hq, alike = a.Hq == a.Hkv;
  const int L = a.Hq * HD, own = (is_k ? hh - a.Hq : hh) * HD;
  // q heads get the mean of k, k heads that of q; as many of one as of the
  // other: each head its own pair's
  const int first = alike ? own : (is_k ? 0 : L), step = alike ? L : HD, heads = alike ? 2 : (is_k ? a.Hq : a.Hkv);
  const float weight = alike ? 0.5f : 0.5f / static_cast<float>(heads);
  for (int i = threadIdx.x; i < 8 * HD; i += threads) {
    const int r = i / (HD / 2), d = 2 * (i % (HD / 2)), n = n0 + r;
    if (n >= a.N) continue;
    const T* row = static_cast<const T*>(a.qkv) + n * a.qkv_rs + first + d;
    float s0 = 0.f, s1 = 0.f;
    for (int h = 0; h < heads; h += 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const Pair<T> x(row + min(h + j, heads - 1) * step);
        const float on = h + j < heads ? 1.f : 0.f;
        s0 = fmaf(x.v[0], on, s0);
        s1 = fmaf(x.v[1], on, s1);
      }
    }
    mean[d][r] = s0 * weight;
    mean[d + 1][r] = s1 * weight;
  }
}

// What the end of the chain reads, for one request and head by 16 neighbouring
// lanes (lane i: the channel pairs i, i + 16, ...): loaded without a branch or a
// wait before the convs' sums are there.
template <typename T, int HD>
struct Tail {
  static constexpr int PP = (HD / 2 + 15) / 16;
  int p;
  float c[PP], s[PP], gain;
  uint32_t v[PP][sizeof(T) / 2];  // a pair as it lies in memory
  int64_t slot;

  __device__ __forceinline__ void load(const DecodeArgs& a, int n, int pos, int hh, int lane) {
    p = pos;
    const bool is_k = hh >= a.Hq;
    const int head = is_k ? hh - a.Hq : 0, K = a.Hkv * HD, at = a.Hq * HD + K;
    const T *now = row_at<T>(a, n, p, 0), *before = p > 0 ? row_at<T>(a, n, p, 1) : now;
    const bool shift = a.flags & HYDRA_CCGQA_VALUE_SHIFT;
    gain = is_k && (a.flags & HYDRA_CCGQA_QK_NORM) ? to_f32(*static_cast<const T*>(a.temp)) : 1.f;
    slot = a.slots[n];
#pragma unroll
    for (int k = 0; k < PP; ++k) {
      const int i = min(lane + 16 * k, HD / 2 - 1), ch = head * HD + 2 * i;
      c[k] = 1.f;
      s[k] = 0.f;
      if (a.flags & HYDRA_CCGQA_ROPE) rope_at(a, max(p, 0), i, c[k], s[k]);
      const bool old = shift && ch >= K / 2;  // K / 2 is a multiple of 8: no pair straddles it
      const uint32_t* lo = reinterpret_cast<const uint32_t*>((old ? before : now) + at + ch);
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(T) / 2); ++w) v[k][w] = old && p <= 0 ? 0u : lo[w];
    }
  }

  // y(d): conv2's channel d; mean(d): its QK-mean term.
  template <typename Y, typename M>
  __device__ __forceinline__ void store(const DecodeArgs& a, int n, int hh, int lane, Y y, M mean) {
    const bool is_k = hh >= a.Hq, add = a.flags & HYDRA_CCGQA_QK_MEAN;
    const int head = is_k ? hh - a.Hq : hh;
    float z[PP][2], sum = 0.f;
#pragma unroll
    for (int k = 0; k < PP; ++k) {
      const int i = min(lane + 16 * k, HD / 2 - 1);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        z[k][e] = y(2 * i + e) + (add ? mean(2 * i + e) : 0.f);
        sum = fmaf(z[k][e], lane + 16 * k < HD / 2 ? z[k][e] : 0.f, sum);
      }
    }
    if (a.flags & HYDRA_CCGQA_QK_NORM) gain /= fmaxf(sqrtf(wave_sum<16>(sum)), 1e-12f);  // F.normalize's eps
    if (p < 0 && is_k) return;
    T *out, *vout = nullptr;
    if (is_k) {
      const int64_t page = slot >> a.shift, r = slot & ((int64_t(1) << a.shift) - 1);
      out = static_cast<T*>(a.kp) + page * a.kps[0] + head * a.kps[1] + r * a.kps[2];
      vout = static_cast<T*>(a.vp) + page * a.vps[0] + head * a.vps[1] + r * a.vps[2];
    } else {
      out = static_cast<T*>(a.q) + (static_cast<int64_t>(n) * a.Hq + head) * HD;
    }
#pragma unroll
    for (int k = 0; k < PP; ++k) {
      const int i = lane + 16 * k;
      if (i >= HD / 2) continue;
      const float x0 = z[k][0] * gain, x1 = z[k][1] * gain;
      out[2 * i] = from_f32<T>(p < 0 ? 0.f : x0 * c[k] - x1 * s[k]);
      out[2 * i + 1] = from_f32<T>(p < 0 ? 0.f : x0 * s[k] + x1 * c[k]);
      if (is_k) {
        T pair[2];
        __builtin_memcpy(pair, v[k], sizeof(pair));
        vout[2 * i] = pair[0];
        vout[2 * i + 1] = pair[1];
      }
    }
  }
};

// A workgroup computes one head of 16 requests over `span` blocks of 16 conv1
// channels (all of them, or a part: blockIdx.z); a wave takes a block at a time,
// conv1's channels there and their share of conv2 at once, and the waves' y2 are
// added up in LDS.  Parts leave their sums in `part` [split][head][tile][16][HD],
// which decode_join_kernel adds in order.  Weights come from L2 (each head
// reads all of conv1's); bound by the chain position -> rows -> convs -> norm:
// one request, 4/1 heads of 64, 7.6 us; 256, 8/2 heads of 64, 19.3 us, where 160
// workgroups on 256 CUs go through two channel blocks a wave and draw 65 MB from
// L2, 0.4 MB each at 21 GB/s, less than a CU can.
template <typename T, int HB, bool TILED>
__global__ __launch_bounds__(64 * decode_waves(HB, sizeof(T))) void decode_prep_mfma_kernel(DecodeArgs a) {
  constexpr int HD = HB * 16;
  constexpr int K = sizeof(T) == 2 && HB >= 2 ? 32 : 16, IB = HD / K;
  constexpr int CH = HB * sizeof(T) >= 32 ? IB / 2 : IB;  // operand blocks in flight
  __shared__ float part[decode_waves(HB, sizeof(T))][HD][17], mean[HD][17];
  const int NW = blockDim.x >> 6;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hh = blockIdx.x, n0 = blockIdx.y * 16;
  const bool is_k = hh >= a.Hq;
  const int L = a.Hq * HD, C = is_k ? a.Hkv * HD : L, col0 = is_k ? L : 0, head = is_k ? hh - a.Hq : hh;
  const int begin = blockIdx.z * a.span, end = min(C / 16, begin + a.span);
  if (begin >= end) return;
  const bool whole = C / 16 <= a.span;
  const Weights<T, K, TILED> w1(a.w[is_k ? 2 : 0], C, HD);
  const Weights<T, 16, TILED> w2(a.w[is_k ? 3 : 1], C, C);
  const int n = n0 + (lane & 15), g = lane >> 4;
  const int p = active_position(a, n);
  if (whole) mean_fill<T, HD>(a, n0, hh, 64 * NW, mean);
  // byte offsets of the rows 4 .. 1 tokens back in the ring, and of the newest
  // (columns of no request read the first row: nothing is made of them)
  uint32_t xo[5];
  {
    const int W = L + 2 * a.Hkv * HD, now = p < 0 ? 0 : p % a.R, m = p < 0 ? 0 : n;
    const uint32_t in_row = (col0 + K / 4 * g) * sizeof(T);
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const int at = now - (4 - o);
      xo[o] = static_cast<uint32_t>(m * a.R + (at < 0 ? at + a.R : at)) * static_cast<uint32_t>(W * sizeof(T)) + in_row;
    }
    xo[4] = static_cast<uint32_t>(m) * static_cast<uint32_t>(a.qkv_rs * sizeof(T)) + in_row;
  }
  const bool young = __any(p >= 0 && p < 4);  // rows before the sequence began count as zero
  Tail<T, HD> tail;
  const int p_tail = __shfl(p, tid >> 4 & 15);  // lane r has request n0 + r
  const bool finishes = whole && tid < 256 && n0 + (tid >> 4) < a.N;
  if (finishes) tail.load(a, n0 + (tid >> 4), p_tail, hh, tid & 15);
  f32x4_t y2[HB];
#pragma unroll
  for (int ob = 0; ob < HB; ++ob) y2[ob] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int cb = begin + wave; cb < end; cb += NW) {  // conv1's output channels 16 cb ..
    const int group = cb / HB;
    f32x4_t y1[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) y1[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i0 = 0; i0 < IB; i0 += CH) {
      Frag<T, K> w1f[CH][3], xf[CH][5];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int64_t in_group = static_cast<int64_t>(group * HD + (i0 + i) * K) * static_cast<int64_t>(sizeof(T));
#pragma unroll
        for (int t = 0; t < 3; ++t) w1f[i][t] = w1(t, cb, i0 + i);
#pragma unroll
        for (int o = 0; o < 5; ++o)
          xf[i][o] = *reinterpret_cast<const Frag<T, K>*>(static_cast<const char*>(o == 4 ? a.qkv : a.ring) + in_group +
                                                          xo[o]);
      }
      if (young) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int o = 0; o < 4; ++o)
            if (p < 4 - o) xf[i][o] = Frag<T, K>{};
      }
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int t = 0; t < 3; ++t)
#pragma unroll
          for (int j = 0; j < 3; ++j) y1[j] = mma<T, K>(w1f[i][t], xf[i][j + t], y1[j]);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const Y1<T> y(y1[j]);
#pragma unroll
      for (int ob = 0; ob < HB; ++ob) y2[ob] = y.times(w2(j, head * HB + ob, cb), y2[ob]);
    }
  }
#pragma unroll
  for (int ob = 0; ob < HB; ++ob)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][ob * 16 + 4 * g + r][lane & 15] = y2[ob][r];
  __syncthreads();
  for (int i = tid; i < HD * 16; i += 64 * NW) {
    const int d = i % HD, r = i / HD;
    float s = part[0][d][r];
#pragma unroll 4
    for (int w = 1; w < NW; ++w) s += part[w][d][r];
    if (whole) part[0][d][r] = s;
    else a.part[((static_cast<int64_t>(blockIdx.z) * gridDim.x + hh) * gridDim.y + blockIdx.y) * 16 * HD + i] = s;
  }
  if (whole) {
    __syncthreads();
    const int r = tid >> 4;
    if (finishes)
      tail.store(a, n0 + r, hh, tid & 15, [&](int d) { return part[0][d][r]; }, [&](int d) { return mean[d][r]; });
  }
  if (hh == 0 && blockIdx.z == 0)
    for (int r = wave; r < 16; r += NW) keep_row16(a, n0 + r, __shfl(p, r), lane, sizeof(T));
}

// The parts of the heads that took more than one workgroup, added in order by
// 1024 threads, eight loads of an element at a time; then the chain's end.
template <typename T, int HB>
__global__ __launch_bounds__(1024) void decode_join_kernel(DecodeArgs a) {
  constexpr int HD = HB * 16;
  __shared__ float mean[HD][17], sum[HD][17];
  const int tid = threadIdx.x, hh = blockIdx.x, n0 = blockIdx.y * 16, r = tid >> 4, n = n0 + r;
  const int C = (hh < a.Hq ? a.Hq : a.Hkv) * HD, splits = (C / 16 + a.span - 1) / a.span;
  if (splits == 1) return;
  const bool finishes = tid < 256 && n < a.N;
  Tail<T, HD> tail;
  if (finishes) tail.load(a, n, active_position(a, n), hh, tid & 15);
  mean_fill<T, HD>(a, n0, hh, 1024, mean);
  const int64_t step = static_cast<int64_t>(gridDim.x) * gridDim.y * 16 * HD;
  const float* part = a.part + (static_cast<int64_t>(hh) * gridDim.y + blockIdx.y) * 16 * HD;
  for (int i = tid; i < 16 * HD; i += 1024) {
    float s = 0.f;
    for (int z = 0; z < splits; z += 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(part[min(z + j, splits - 1) * step + i], z + j < splits ? 1.f : 0.f, s);
    }
    sum[i % HD][i / HD] = s;
  }
  __syncthreads();
  if (finishes)
    tail.store(a, n, hh, tid & 15, [&](int d) { return sum[d][r]; }, [&](int d) { return mean[d][r]; });
}

constexpr int64_t kDecodeRequests = 65535, kDecodeHeads = 4096;  // of a call

bool decode_mfma_size(int64_t hd, int64_t ks, int flags) {
  return (flags & HYDRA_CCGQA_CONVS) && ks == 3 && (hd == 16 || hd == 32 || hd == 64 || hd == 128);
}

template <typename T>
int launch_decode(DecodeArgs a, hipStream_t st) {
  const int L = a.Hq * a.hd, W = L + 2 * a.Hkv * a.hd;
  const int need = 16 / static_cast<int>(sizeof(T));
  // rows and weights that 16-byte loads take
  bool vec = a.qkv_rs % need == 0 && W % need == 0 && aligned16(a.qkv) && aligned16(a.ring);
  for (const void* w : a.w) vec = vec && aligned16(w);
  bool mfma = vec && decode_mfma_size(a.hd, a.ks, a.flags);
  // 32-bit byte offsets of rows
  mfma = mfma && static_cast<int64_t>(a.N) * a.R * W * sizeof(T) < (int64_t(1) << 32) &&
         a.N * a.qkv_rs * static_cast<int64_t>(sizeof(T)) < (int64_t(1) << 32);
  const bool tiled = a.flags & HYDRA_CCGQA_W_TILED;
  // the matrix form's: other sizes may have no block of 16 channels
  const DecodePlan plan = mfma ? decode_plan(a.N, a.Hq, a.Hkv, a.hd, sizeof(T), tiled) : DecodePlan{};
  a.span = plan.span;
  const dim3 tiles(static_cast<unsigned>(a.Hq + a.Hkv), static_cast<unsigned>((a.N + 15) / 16));
  const dim3 parts(tiles.x, tiles.y, static_cast<unsigned>(plan.splits));
  // More workgroups than CUs: of half as many waves two share a CU (512 requests,
  // 8/8 heads of 32: 15.8 us with 16 waves, 13.9 with 8; no more than CUs, 256
  // requests, 4/1 heads of 64: 12.1 and 13.4).
  const bool shared = static_cast<int64_t>(tiles.x) * tiles.y > device_cus();
  const int threads = 64 * (shared && plan.waves > 8 ? 8 : plan.waves);
#define HYDRA_DECODE(HB)                                                                          \
  {                                                                                               \
    if constexpr (sizeof(T) == 2) {                                                               \
      if (tiled) decode_prep_mfma_kernel<T, HB, true><<<parts, threads, 0, st>>>(a);              \
    }                                                                                             \
    if (!tiled) decode_prep_mfma_kernel<T, HB, false><<<parts, threads, 0, st>>>(a);              \
    if (plan.splits > 1) decode_join_kernel<T, HB><<<tiles, 1024, 0, st>>>(a);                    \
  }
  if (mfma && a.hd == 16) HYDRA_DECODE(1)
  else if (mfma && a.hd == 32) HYDRA_DECODE(2)
  else if (mfma && a.hd == 64) HYDRA_DECODE(4)
  else if (mfma) HYDRA_DECODE(8)
  else {
    if (tiled)
      return fail(HYDRA_ERR_UNSUPPORTED, "ccgqa_decode_prep: tiled weights need the matrix-core form");
    const size_t y1 = a.flags & HYDRA_CCGQA_CONVS ? static_cast<size_t>(a.ks) * std::max(a.Hq, a.Hkv) * a.hd : 0;
    const size_t lds = sizeof(float) * (y1 + a.hd);
    if (lds > 64 * 1024)
      return fail(HYDRA_ERR_UNSUPPORTED, "ccgqa_decode_prep: conv taps times channels above 16384 need head_dim 16, "
                                         "32, 64 or 128 and three taps");
    const dim3 grid(tiles.x, static_cast<unsigned>(a.N));
    if (vec && a.hd % need == 0) decode_prep_generic_kernel<T, true><<<grid, kGenericThreads, lds, st>>>(a);
    else decode_prep_generic_kernel<T, false><<<grid, kGenericThreads, lds, st>>>(a);
  }
#undef HYDRA_DECODE
  return check_launch("ccgqa_decode_prep");
}

// The last `keep` rows of prompts into the ring: qkv [M, S, W], prompt m being
// request r = rows[m], row s if lengths[r] - keep <= s < lengths[r] to
// ring[r][s % R].  The workgroups from `keep` on set the rows past the prompt's
// end to zero (none of them is kept): a matrix product over a tile would
// multiply what lies there by a weight of 0, and 0 * inf is NaN.  16 prompts of 1024
// rows of 768 bytes: 3.8 us, 7.3 with half of them cleared.
template <typename T>
__global__ __launch_bounds__(256) void ring_fill_kernel(T* qkv, int64_t bs, int64_t rs, T* ring, const int64_t* rows,
                                                        const int* lengths, int N, int R, int W, int S, int keep) {
  const int m = blockIdx.y, b = blockIdx.x;
  const int64_t row = rows ? rows[m] : m;
  if (row < 0 || row >= N) return;
  const int len = lengths[row];
  if (len <= 0 || len > S) return;
  T* x = qkv + m * bs;
  if (b < keep) {
    const int s = len - 1 - b;
    if (s < 0) return;
    T* to = ring + (row * R + s % R) * W;
    for (int c = threadIdx.x; c < W; c += 256) to[c] = x[s * rs + c];
  } else {
    const int step = gridDim.x - keep;
    for (int64_t s = static_cast<int64_t>(len) + b - keep; s < S; s += step)
      for (int c = threadIdx.x; c < W; c += 256) x[s * rs + c] = from_f32<T>(0.f);
  }
}

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int64_t hydra_ccgqa_decode_prep_workspace(int64_t N, int64_t Hq, int64_t Hkv, int64_t hd, int64_t conv_ks,
                                                     int flags, int dtype) {
  const int e = dtype_size(dtype);
  if (N <= 0 || Hq <= 0 || Hkv <= 0 || e == 0 || !decode_mfma_size(hd, conv_ks, flags)) return 0;
  if (N > kDecodeRequests || Hq > kDecodeHeads || Hkv > Hq) return 0;  // which hydra_ccgqa_decode_prep refuses
  const int splits = decode_plan(N, Hq, Hkv, hd, e, flags & HYDRA_CCGQA_W_TILED).splits;
  return splits == 1 ? 0 : 4 * static_cast<int64_t>(splits) * (Hq + Hkv) * ((N + 15) / 16) * 16 * hd;
}

extern "C" int hydra_ccgqa_decode_prep(const void* qkv, int64_t qkv_rs, void* ring, int64_t R, const int* positions,
                                       const int64_t* slots, const void* wq1, const void* wq2, const void* wk1,
                                       const void* wk2, const void* temperature, const void* cos, const void* sin,
                                       int64_t cs_rs, int64_t rope_rows, void* q, void* k_pages, void* v_pages,
                                       const int64_t* kp_st, const int64_t* vp_st, int64_t pages, int64_t page_size,
                                       int64_t N, int64_t Hq, int64_t Hkv, int64_t hd, int64_t conv_ks, int flags,
                                       int dtype, void* workspace, int64_t workspace_size, void* stream) {
  constexpr int known = HYDRA_CCGQA_CONVS | HYDRA_CCGQA_QK_MEAN | HYDRA_CCGQA_VALUE_SHIFT | HYDRA_CCGQA_QK_NORM |
                        HYDRA_CCGQA_ROPE | HYDRA_CCGQA_W_TILED | HYDRA_CCGQA_ROPE_BF16;
  HYDRA_REQUIRE((flags & ~known) == 0, "ccgqa_decode_prep: unknown flag");
  HYDRA_REQUIRE(N >= 0 && Hq >= 1 && Hkv >= 1 && hd >= 2 && pages >= 1, "ccgqa_decode_prep: bad size");
  HYDRA_REQUIRE(hd % 2 == 0, "ccgqa_decode_prep: head_dim must be even");
  HYDRA_REQUIRE(Hq % Hkv == 0, "ccgqa_decode_prep: n_heads must be a multiple of n_kv_heads");
  HYDRA_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
                "ccgqa_decode_prep: page_size must be a power of two in [16, 4096]");
  const bool convs = flags & HYDRA_CCGQA_CONVS;
  HYDRA_REQUIRE(!convs || (conv_ks >= 1 && conv_ks <= 16), "ccgqa_decode_prep: conv taps must be in [1, 16]");
  const int64_t back = std::max<int64_t>(convs ? 2 * (conv_ks - 1) : 0, flags & HYDRA_CCGQA_VALUE_SHIFT ? 1 : 0);
  HYDRA_REQUIRE(R > back && R < (1 << 20), "ccgqa_decode_prep: the ring must hold more rows than a token looks back");
  HYDRA_REQUIRE(N <= kDecodeRequests && Hq <= kDecodeHeads && hd <= 4096 && pages < (int64_t(1) << 31),
                "ccgqa_decode_prep: too large");
  const int64_t W = (Hq + 2 * Hkv) * hd;
  HYDRA_REQUIRE(qkv_rs >= W || N <= 1, "ccgqa_decode_prep: row stride < L + 2K");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "ccgqa_decode_prep: unknown dtype");
  HYDRA_REQUIRE(!(flags & HYDRA_CCGQA_W_TILED) || (convs && dtype != HYDRA_F32 && (Hkv * hd) % 32 == 0),
                "ccgqa_decode_prep: tiled weights are 16-bit, of whole blocks of 32 channels");
  if (N == 0) return HYDRA_OK;
  HYDRA_REQUIRE(qkv && ring && positions && slots && q && k_pages && v_pages && kp_st && vp_st,
                "ccgqa_decode_prep: null pointer");
  HYDRA_REQUIRE(!convs || (wq1 && wq2 && wk1 && wk2), "ccgqa_decode_prep: convs need their four weights");
  HYDRA_REQUIRE(!(flags & HYDRA_CCGQA_QK_NORM) || temperature, "ccgqa_decode_prep: QK-norm needs temperature");
  HYDRA_REQUIRE(!(flags & HYDRA_CCGQA_ROPE) || (cos && sin && cs_rs >= hd / 2 && rope_rows >= 1),
                "ccgqa_decode_prep: RoPE needs cos/sin");
  HYDRA_REQUIRE(kp_st[3] == 1 && vp_st[3] == 1, "ccgqa_decode_prep: pages need rows of unit stride");
  const int64_t need = hydra_ccgqa_decode_prep_workspace(N, Hq, Hkv, hd, conv_ks, flags, dtype);
  HYDRA_REQUIRE(workspace_size >= need && (need == 0 || (workspace && aligned16(workspace))),
                "ccgqa_decode_prep: workspace too small");
  DecodeArgs a{};
  a.qkv = qkv;
  a.qkv_rs = qkv_rs;
  a.ring = ring;
  a.positions = positions;
  a.slots = slots;
  a.w[0] = wq1;
  a.w[1] = wq2;
  a.w[2] = wk1;
  a.w[3] = wk2;
  a.temp = temperature;
  a.cos = cos;
  a.sin = sin;
  a.cs_rs = cs_rs;
  a.rope_rows = static_cast<int>(std::min<int64_t>(rope_rows, INT32_MAX));
  a.q = q;
  a.kp = k_pages;
  a.vp = v_pages;
  for (int i = 0; i < 3; ++i) {
    a.kps[i] = kp_st[i];
    a.vps[i] = vp_st[i];
  }
  a.limit = pages * page_size;
  a.N = static_cast<int>(N);
  a.R = static_cast<int>(R);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.hd = static_cast<int>(hd);
  a.ks = static_cast<int>(conv_ks);
  a.shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  a.flags = flags;
  a.part = static_cast<float*>(workspace);
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int { return launch_decode<T>(a, st); });
}

extern "C" int hydra_ccgqa_ring_fill(void* qkv, int64_t qkv_bs, int64_t qkv_rs, void* ring, const int64_t* rows,
                                     const int* lengths, int64_t M, int64_t S, int64_t W, int64_t N, int64_t R,
                                     int64_t keep, int clear, int dtype, void* stream) {
  HYDRA_REQUIRE(M >= 0 && S >= 1 && W >= 1 && N >= 1 && R >= 1 && keep >= 0, "ccgqa_ring_fill: bad size");
  HYDRA_REQUIRE(keep <= R, "ccgqa_ring_fill: more rows than the ring holds");
  HYDRA_REQUIRE(M <= 65535 && S < (int64_t(1) << 31) && W < (int64_t(1) << 31) && N < (int64_t(1) << 31) &&
                    R < (1 << 20),
                "ccgqa_ring_fill: too large");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "ccgqa_ring_fill: unknown dtype");
  // workgroups of a prompt that clear: one a row, up to 128
  const int64_t past = clear ? std::min<int64_t>(S, 128) : 0;
  if (M == 0 || keep + past == 0) return HYDRA_OK;
  HYDRA_REQUIRE(qkv && ring && lengths, "ccgqa_ring_fill: null pointer");
  HYDRA_REQUIRE(rows || M <= N, "ccgqa_ring_fill: more prompts than rows");
  const dim3 grid(static_cast<unsigned>(keep + past), static_cast<unsigned>(M));
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    ring_fill_kernel<T><<<grid, 256, 0, st>>>(static_cast<T*>(qkv), qkv_bs, qkv_rs, static_cast<T*>(ring), rows,
                                              lengths, static_cast<int>(N), static_cast<int>(R), static_cast<int>(W),
                                              static_cast<int>(S), static_cast<int>(keep));
    return check_launch("ccgqa_ring_fill");
  });
}
