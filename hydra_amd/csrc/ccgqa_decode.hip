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
// fp32 throughout, one rounding at the end; the MFMA form carries y1 into conv2 as
// two 16-bit terms (16 significant bits for bf16, 22 for fp16).
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

// Channel c of v.
template <typename T>
__device__ __forceinline__ T value_at(const DecodeArgs& a, int n, int p, int c) {
  const int K = a.Hkv * a.hd, at = a.Hq * a.hd + K;
  const T* row = row_at<T>(a, n, p, 0);
  if (!(a.flags & HYDRA_CCGQA_VALUE_SHIFT) || c < K / 2) return row[at + c];
  return p > 0 ? row_at<T>(a, n, p, 1)[at + c] : from_f32<T>(0.f);
}

// Everything after the convs, for one request and head, by LANES neighbouring
// lanes of a wave (lane i of them has the channel pairs i, i + LANES, ...);
// y(d) gives conv2's channel d.
template <typename T, int LANES, typename Y>
__device__ __forceinline__ void finish(const DecodeArgs& a, int n, int p, int hh, int lane, Y y) {
  const bool is_k = hh >= a.Hq;
  const int head = is_k ? hh - a.Hq : hh, pairs = a.hd / 2;
  T* qrow = is_k ? nullptr : static_cast<T*>(a.q) + (static_cast<int64_t>(n) * a.Hq + head) * a.hd;
  if (p < 0) {
    if (!is_k)
      for (int d = lane; d < a.hd; d += LANES) qrow[d] = from_f32<T>(0.f);
    return;
  }
  const T* row = row_at<T>(a, n, p, 0);
  const bool mean = a.flags & HYDRA_CCGQA_QK_MEAN;
  float gain = 1.f;
  if (a.flags & HYDRA_CCGQA_QK_NORM) {
    float s = 0.f;
    for (int i = lane; i < pairs; i += LANES)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float v = y(2 * i + e) + (mean ? mean_term<T>(a, row, hh, 2 * i + e) : 0.f);
        s = fmaf(v, v, s);
      }
    s = wave_sum<LANES>(s);
    gain = 1.f / fmaxf(sqrtf(s), 1e-12f);  // F.normalize's eps
    if (is_k) gain *= to_f32(*static_cast<const T*>(a.temp));
  }
  T *out = qrow, *vout = nullptr;
  if (is_k) {
    const int64_t slot = a.slots[n], page = slot >> a.shift, r = slot & ((int64_t(1) << a.shift) - 1);
    out = static_cast<T*>(a.kp) + page * a.kps[0] + head * a.kps[1] + r * a.kps[2];
    vout = static_cast<T*>(a.vp) + page * a.vps[0] + head * a.vps[1] + r * a.vps[2];
  }
  for (int i = lane; i < pairs; i += LANES) {
    float v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      v[e] = (y(2 * i + e) + (mean ? mean_term<T>(a, row, hh, 2 * i + e) : 0.f)) * gain;
    if (a.flags & HYDRA_CCGQA_ROPE) {
      const int64_t at = static_cast<int64_t>(p) * a.cs_rs + i;
      float c, s;
      if (a.flags & HYDRA_CCGQA_ROPE_BF16) {
        c = to_f32(static_cast<const bf16*>(a.cos)[at]);
        s = to_f32(static_cast<const bf16*>(a.sin)[at]);
      } else {
        c = static_cast<const float*>(a.cos)[at];
        s = static_cast<const float*>(a.sin)[at];
      }
      const float x0 = v[0], x1 = v[1];
      v[0] = x0 * c - x1 * s;
      v[1] = x0 * s + x1 * c;
    }
    out[2 * i] = from_f32<T>(v[0]);
    out[2 * i + 1] = from_f32<T>(v[1]);
  }
  if (is_k)
    for (int d = lane; d < a.hd; d += LANES) vout[d] = value_at<T>(a, n, p, head * a.hd + d);
}

template <typename T>
__device__ __forceinline__ void keep_row(const DecodeArgs& a, int n, int p, int tid, int threads) {
  if (p < 0) return;
  const int W = (a.Hq + 2 * a.Hkv) * a.hd;
  const T* from = row_at<T>(a, n, p, 0);
  T* to = static_cast<T*>(a.ring) + (static_cast<int64_t>(n) * a.R + p % a.R) * W;
  for (int c = tid; c < W; c += threads) to[c] = from[c];
}

// Any head_dim, taps and flags: one workgroup per request and head on the
// VALU, y1 in LDS as [ks][C] floats, then y2 [hd].
template <typename T>
__global__ __launch_bounds__(256) void decode_prep_generic_kernel(DecodeArgs a) {
  extern __shared__ float sm[];
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
    for (int i = tid; i < a.ks * C; i += 256) {
      const int j = i / C, c = i - j * C, g0 = c / hd * hd;
      float s = 0.f;
      for (int t = 0; t < a.ks; ++t) {
        const int back = 2 * (a.ks - 1) - j - t;
        if (back > p) continue;
        const T* x = row_at<T>(a, n, p, back) + col0 + g0;
        const T* w = w1 + (static_cast<int64_t>(t) * C + c) * hd;
        for (int e = 0; e < hd; ++e) s = fmaf(to_f32(w[e]), to_f32(x[e]), s);
      }
      sm[i] = s;
    }
    __syncthreads();
    for (int d = wave; d < hd; d += 4) {
      float s = 0.f;
      for (int j = 0; j < a.ks; ++j) {
        const T* w = w2 + (static_cast<int64_t>(j) * C + head * hd + d) * C;
        for (int c = lane; c < C; c += 64) s = fmaf(to_f32(w[c]), sm[j * C + c], s);
      }
      s = wave_sum(s);
      if (lane == 0) y2[d] = s;
    }
  } else if (p >= 0) {
    const T* x = row_at<T>(a, n, p, 0) + col0 + head * hd;
    for (int d = tid; d < hd; d += 256) y2[d] = to_f32(x[d]);
  }
  __syncthreads();
  if (wave == 0) finish<T, 64>(a, n, p, hh, lane, [&](int d) { return y2[d]; });
  if (hh == 0) keep_row<T>(a, n, p, tid, 256);
}

// ---- matrix-core form: three taps, head_dim a multiple of 16 ----------------
// A lane's four neighbouring values of an operand of v_mfma_f32_16x16x16 (row
// or column lane & 15, k = 4 (lane >> 4) + i), or of four v_mfma_f32_16x16x4
// in fp32 (the i-th takes element i: k is a name that both operands share).
// The result's lane holds column lane & 15, rows 4 (lane >> 4) + i: what the next
// product wants as its operand, so y1 goes from conv1 to conv2 in registers.
template <typename T>
using Frag = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;

template <typename T>
__device__ __forceinline__ f32x4_t mma(Frag<T> a, Frag<T> b, f32x4_t c) {
  if constexpr (std::is_same<T, float>::value) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
  } else if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c,
                                                     0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a), __builtin_bit_cast(f16x4_t, b), c, 0,
                                                 0, 0);
  }
}

// c += a y for an fp32 y: one product of fp32, two of a 16-bit type (the
// rounded value and what it leaves).
template <typename T>
struct Split {
  Frag<T> hi, lo;
  __device__ __forceinline__ explicit Split(f32x4_t y) {
    if constexpr (sizeof(T) == 4) {
      hi = make_float4(y[0], y[1], y[2], y[3]);
    } else {
      float rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float h = to_f32(from_f32<T>(y[i]));
        rest[i] = fabsf(h) == INFINITY ? 0.f : y[i] - h;
      }
      hi = make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
      lo = make_uint2(pack2<T>(rest[0], rest[1]), pack2<T>(rest[2], rest[3]));
    }
  }
  __device__ __forceinline__ f32x4_t times(Frag<T> a, f32x4_t c) const {
    c = mma<T>(a, hi, c);
    if constexpr (sizeof(T) == 2) c = mma<T>(a, lo, c);
    return c;
  }
};

// Operand block (tap t, output channels 16 ob .., input channels 16 ib ..) of a
// weight [3][O][I], or of its MFMA-tiled order [3][O/32][I/16][2][32][8].
template <typename T>
__device__ __forceinline__ Frag<T> weight_frag(const void* w, bool tiled, int O, int I, int t, int ob, int ib) {
  const int lane = threadIdx.x & 63, g = lane >> 4, o = ob * 16 + (lane & 15);
  int64_t at = static_cast<int64_t>(t) * O * I;
  if (tiled) at += (static_cast<int64_t>(o >> 5) * (I >> 4) + ib) * 512 + ((g >> 1) * 32 + (o & 31)) * 8 + (g & 1) * 4;
  else at += static_cast<int64_t>(o) * I + ib * 16 + 4 * g;
  return *reinterpret_cast<const Frag<T>*>(static_cast<const T*>(w) + at);
}

constexpr int decode_waves(int hb) { return hb <= 4 ? 8 : 4; }

// A workgroup computes one head of 16 requests: its waves take the input
// groups (C / hd of them) in turn, conv1 of a group's 16 channels at a time and
// its share of conv2 at once, and add up their y2 in LDS.  Weights come from L2
// (every workgroup of a head reads the same); bound by that stream and the
// chain of the loads: 5 to 8 us for up to 256 requests.
template <typename T, int HB>
__global__ __launch_bounds__(64 * decode_waves(HB)) void decode_prep_mfma_kernel(DecodeArgs a) {
  constexpr int NW = decode_waves(HB), HD = HB * 16;
  __shared__ float part[NW][HD][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hh = blockIdx.x, n0 = blockIdx.y * 16;
  const bool is_k = hh >= a.Hq, tiled = a.flags & HYDRA_CCGQA_W_TILED;
  const int L = a.Hq * HD, C = is_k ? a.Hkv * HD : L, col0 = is_k ? L : 0, head = is_k ? hh - a.Hq : hh;
  const void *w1 = a.w[is_k ? 2 : 0], *w2 = a.w[is_k ? 3 : 1];
  const int n = n0 + (lane & 15), g = lane >> 4;
  const int p = active_position(a, n);
  const T* x[5];  // the rows 4 .. 0 tokens back
#pragma unroll
  for (int o = 0; o < 5; ++o)
    x[o] = (p >= 4 - o ? row_at<T>(a, n, p, 4 - o) : static_cast<const T*>(a.qkv)) + col0 + 4 * g;
  f32x4_t y2[HB];
#pragma unroll
  for (int ob = 0; ob < HB; ++ob) y2[ob] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int cb = wave; cb < C / 16; cb += NW) {  // conv1's output channels 16 cb ..
    const int group = cb / HB;
    f32x4_t y1[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) y1[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ib = 0; ib < HB; ++ib) {
      Frag<T> xf[5], wf[3];
#pragma unroll
      for (int o = 0; o < 5; ++o) {
        xf[o] = *reinterpret_cast<const Frag<T>*>(x[o] + group * HD + ib * 16);
        if (p < 4 - o) xf[o] = Frag<T>{};  // before the sequence began, or no request
      }
#pragma unroll
      for (int t = 0; t < 3; ++t) wf[t] = weight_frag<T>(w1, tiled, C, HD, t, cb, ib);
#pragma unroll
      for (int j = 0; j < 3; ++j)
#pragma unroll
        for (int t = 0; t < 3; ++t) y1[j] = mma<T>(wf[t], xf[j + t], y1[j]);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const Split<T> y(y1[j]);
#pragma unroll
      for (int ob = 0; ob < HB; ++ob)
        y2[ob] = y.times(weight_frag<T>(w2, tiled, C, C, j, head * HB + ob, cb), y2[ob]);
    }
  }
#pragma unroll
  for (int ob = 0; ob < HB; ++ob)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][ob * 16 + 4 * g + r][lane & 15] = y2[ob][r];
  __syncthreads();
  for (int i = tid; i < HD * 16; i += 64 * NW) {
    const int d = i >> 4, r = i & 15;
    float s = part[0][d][r];
#pragma unroll
    for (int w = 1; w < NW; ++w) s += part[w][d][r];
    part[0][d][r] = s;
  }
  __syncthreads();
  // 16 lanes a request
  for (int r = tid >> 4; r < 16; r += 4 * NW) {
    const int m = n0 + r;
    if (m < a.N) finish<T, 16>(a, m, active_position(a, m), hh, tid & 15, [&](int d) { return part[0][d][r]; });
  }
  if (hh == 0)
    for (int r = wave; r < 16; r += NW)
      if (n0 + r < a.N) keep_row<T>(a, n0 + r, active_position(a, n0 + r), lane, 64);
}

template <typename T>
int launch_decode(const DecodeArgs& a, hipStream_t st) {
  const int W = (a.Hq + 2 * a.Hkv) * a.hd;
  const int need = 16 / static_cast<int>(sizeof(T));
  // the operands are loaded four values at a time: rows and weights aligned to that
  bool mfma = (a.flags & HYDRA_CCGQA_CONVS) && a.ks == 3 && a.qkv_rs % need == 0 && W % need == 0 &&
              aligned16(a.qkv) && aligned16(a.ring);
  for (const void* w : a.w) mfma = mfma && aligned16(w);
  const dim3 tiles(static_cast<unsigned>(a.Hq + a.Hkv), static_cast<unsigned>((a.N + 15) / 16));
#define HYDRA_DECODE(HB) decode_prep_mfma_kernel<T, HB><<<tiles, 64 * decode_waves(HB), 0, st>>>(a)
  if (mfma && a.hd == 16) HYDRA_DECODE(1);
  else if (mfma && a.hd == 32) HYDRA_DECODE(2);
  else if (mfma && a.hd == 64) HYDRA_DECODE(4);
  else if (mfma && a.hd == 128) HYDRA_DECODE(8);
  else {
    if (a.flags & HYDRA_CCGQA_W_TILED)
      return fail(HYDRA_ERR_UNSUPPORTED, "ccgqa_decode_prep: tiled weights need the matrix-core form");
    const size_t lds = sizeof(float) * ((a.flags & HYDRA_CCGQA_CONVS ? static_cast<size_t>(a.ks) * std::max(a.Hq, a.Hkv) * a.hd : 0) + a.hd);
    if (lds > 64 * 1024)
      return fail(HYDRA_ERR_UNSUPPORTED, "ccgqa_decode_prep: conv taps times channels above 16384 need head_dim 16, "
                                         "32, 64 or 128 and three taps");
    decode_prep_generic_kernel<T><<<dim3(static_cast<unsigned>(a.Hq + a.Hkv), static_cast<unsigned>(a.N)), 256, lds,
                                    st>>>(a);
  }
#undef HYDRA_DECODE
  return check_launch("ccgqa_decode_prep");
}

// The last `keep` rows of prompts into the ring: qkv [M, S, W] (strides qs),
// row s of prompt m, if lengths[m] - keep <= s < lengths[m], to
// ring[rows[m]][s % R]; prompts with a length outside [0, S] or a row outside
// the ring leave it as it is.
template <typename T>
__global__ __launch_bounds__(256) void ring_fill_kernel(const T* qkv, int64_t bs, int64_t rs, T* ring,
                                                        const int64_t* rows, const int* lengths, int N, int R, int W,
                                                        int S, int keep) {
  const int m = blockIdx.y, len = lengths[m], s = len - 1 - static_cast<int>(blockIdx.x);
  const int64_t row = rows ? rows[m] : m;
  if (len > S || s < 0 || row < 0 || row >= N) return;
  const T* from = qkv + m * bs + s * rs;
  T* to = ring + (row * R + s % R) * W;
  for (int c = threadIdx.x; c < W; c += 256) to[c] = from[c];
}

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int hydra_ccgqa_decode_prep(const void* qkv, int64_t qkv_rs, void* ring, int64_t R, const int* positions,
                                       const int64_t* slots, const void* wq1, const void* wq2, const void* wk1,
                                       const void* wk2, const void* temperature, const void* cos, const void* sin,
                                       int64_t cs_rs, int64_t rope_rows, void* q, void* k_pages, void* v_pages,
                                       const int64_t* kp_st, const int64_t* vp_st, int64_t pages, int64_t page_size,
                                       int64_t N, int64_t Hq, int64_t Hkv, int64_t hd, int64_t conv_ks, int flags,
                                       int dtype, void* stream) {
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
  HYDRA_REQUIRE(N <= 65535 && Hq <= 4096 && hd <= 4096, "ccgqa_decode_prep: too large");
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
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int { return launch_decode<T>(a, st); });
}

extern "C" int hydra_ccgqa_ring_fill(const void* qkv, int64_t qkv_bs, int64_t qkv_rs, void* ring, const int64_t* rows,
                                     const int* lengths, int64_t M, int64_t S, int64_t W, int64_t N, int64_t R,
                                     int64_t keep, int dtype, void* stream) {
  HYDRA_REQUIRE(M >= 0 && S >= 1 && W >= 1 && N >= 1 && R >= 1 && keep >= 0, "ccgqa_ring_fill: bad size");
  HYDRA_REQUIRE(keep <= R, "ccgqa_ring_fill: more rows than the ring holds");
  HYDRA_REQUIRE(M <= 65535 && S < (int64_t(1) << 31) && W < (int64_t(1) << 31) && N < (int64_t(1) << 31) && R < (1 << 20),
                "ccgqa_ring_fill: too large");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "ccgqa_ring_fill: unknown dtype");
  if (M == 0 || keep == 0) return HYDRA_OK;
  HYDRA_REQUIRE(qkv && ring && lengths, "ccgqa_ring_fill: null pointer");
  HYDRA_REQUIRE(rows || M <= N, "ccgqa_ring_fill: more prompts than rows");
  const dim3 grid(static_cast<unsigned>(keep), static_cast<unsigned>(M));
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    ring_fill_kernel<T><<<grid, 256, 0, st>>>(static_cast<const T*>(qkv), qkv_bs, qkv_rs, static_cast<T*>(ring), rows,
                                              lengths, static_cast<int>(N), static_cast<int>(R), static_cast<int>(W),
                                              static_cast<int>(S), static_cast<int>(keep));
    return check_launch("ccgqa_ring_fill");
  });
}
