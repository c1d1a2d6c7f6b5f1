// Log probabilities of given tokens, the entropy and the top alternatives of
// their rows of logits, forward and backward, gfx950.
//
// With c = log2(e) / temperature, M = max_j x_j, t_j = (x_j - M) c (the
// difference first: right also where every logit is the type's lowest value),
// s = sum 2^t_j, w = sum 2^t_j t_j,
//   logp_j  = (x_j - M) / T - ln2 log2 s, entropy = ln2 (log2 s - w / s),
//   dL/dx_j = 2^t_j (A + B t_j) + ([j = token] g_lp + sum_k [j = i_k] g_k) / T,
//   B = -ln2 g_H / (s T),  A = -(g_lp + sum_k g_k + g_H (H - ln2 log2 s)) / (s T).
// All of it in fp32; gradients are rounded once.  The backward needs M, s and H
// of a row and no sum over it: it is elementwise.
//
// Both directions are bound by HBM: the forward reads a row once and keeps it
// in registers between its maximum and its sums (16-bit values packed), the
// backward reads it once and writes the gradient.  8192 rows of 32000, bf16:
// 108 us, 4.9 TB/s, forward (135 with 20 alternatives) and 190 us, 5.5 TB/s,
// backward.  A few rows take the chain row -> maximum -> sums (-> bound ->
// candidates -> ranks): 16 of 50257, 20 alternatives, 12.1 us.  Where fewer than
// K of 64 groups of lanes hold an allowed logit, or equal ones lead the row, the
// alternatives are taken one by one (see logp_kernel): such rows (12 allowed of
// 50257, or all equal) take 367 us, and a launch with one among them as long.
// Rows start anywhere: a row is taken in the 16-byte pieces of memory that it lies
// in, what is left at its two ends element by element.
#include "common.h"
#include "mod_keys.h"

namespace hydra {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// exp2 of anything below is 0: keeps 0 * t_j a 0 where x_j is -inf.
constexpr float kLowest = -2000.f;
constexpr int kThreads = 512;
constexpr int kMaxTop = 64;
constexpr int kCandidates = 1024;

struct LogpArgs {
  const void* x;
  int64_t rs;
  const int64_t* tokens;
  float *logp, *entropy, *stats;  // stats [rows][2]: M, s
  float* top;                     // [rows][K]
  int64_t* top_tokens;
  int V, K;
  float c, inv_t;  // log2(e) / temperature, 1 / temperature
};

// A row as 16-byte pieces of memory: piece i holds the elements E i - shift + (0 .. E-1);
// pieces [first, last) are whole.  What is left of the row at its two ends, less
// than E elements each, is one element of each of the first 2 E threads.
template <typename T>
struct Pieces {
  static constexpr int E = Vec<T>::N;
  const T* x;
  int shift, first, last;
  int own;  // this thread's element of the ends, or -1
  __device__ __forceinline__ Pieces(const T* row, int V) : x(row) {
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    first = shift > 0 ? 1 : 0;
    last = max((V + shift) / E, first);
    const int head = min(first * E - shift, V);  // elements before the first whole piece
    const int behind = max(last * E - shift, head), tid = threadIdx.x;
    own = tid < E ? (tid < head ? tid : -1) : (tid < 2 * E && behind + tid - E < V ? behind + tid - E : -1);
  }
  __device__ __forceinline__ int element(int piece) const { return piece * E - shift; }
  __device__ __forceinline__ float end() const { return own >= 0 ? to_f32(x[own]) : -INFINITY; }
};

// Sixteen bytes of -inf.
template <typename T>
__device__ __forceinline__ uint4 low_piece() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, bf16>::value ? 0xff80ff80u : 0xfc00fc00u);
  return make_uint4(w, w, w, w);
}

template <int N>
__device__ __forceinline__ float max_of(const float* v) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  return m;
}

// Adds a piece's 2^t and 2^t t to s and w.
template <int N>
__device__ __forceinline__ void add_sums(const float* v, float c, float M, float& s, float& w) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = (v[i] - M) * c, e = __builtin_amdgcn_exp2f(t);
    s += e;
    w = fmaf(e, fmaxf(t, kLowest), w);  // a NaN stays one through e
  }
}

// score_key_asc's inverse (zero for both zeros).
__device__ __forceinline__ float score_of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Order of the alternatives: value down, index up.
__device__ __forceinline__ uint64_t rank_key(float v, int e) {
  return (static_cast<uint64_t>(score_key_asc(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(e));
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int off) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), off), hi = __shfl_xor(static_cast<uint32_t>(v >> 32), off);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The K-th largest of a wave's 64 keys, by their bits from the top: the largest
// value that at least K of them reach.
__device__ __forceinline__ uint32_t kth_of_wave(uint32_t key, int K) {
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = bound | (1u << bit);
    if (__popcll(__ballot(key >= t)) >= K) bound = t;
  }
  return bound;
}

// One row per workgroup.  NCH > 0: its pieces stay in registers, NCH of a
// thread; NCH = 0: read again for the sums (rows of more than 16384 pieces).
//
// Alternatives: 64 groups of 8 lanes keep their maximum; the K-th largest of
// these is a bound that at least K elements reach, and few more (about
// 64 ln(64 / (64 - K)) of them where the order is random: 24 for K = 20).  Only
// threads whose own maximum reaches it look at their pieces again; what they
// find is listed in LDS and ranked against each other.  Where equal values make
// them more than 1024 (masked ones too, where they are the bound), or a NaN leads
// the row, the K best are taken one by one, each by a scan of the row that waits
// for the last one.
template <typename T, int NCH, bool TOP>
__global__ __launch_bounds__(kThreads) void logp_kernel(LogpArgs a) {
  constexpr int E = Vec<T>::N, WAVES = kThreads / 64;
  __shared__ float red[2][WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.rs;
  const Pieces<T> pieces(x, a.V);
  uint4 raw[NCH > 0 ? NCH : 1];
  const int wave_first = __builtin_amdgcn_readfirstlane(pieces.first + (tid & ~63));
  // every whole piece of this thread's
  auto each = [&](auto f) {
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        // the pieces stay packed between the passes: no widened copies kept
        asm volatile("" : "+v"(raw[i].x), "+v"(raw[i].y), "+v"(raw[i].z), "+v"(raw[i].w));
        if (wave_first + i * kThreads >= pieces.last) continue;  // the wave has none here
        float v[E];
        unpack16<T>(raw[i], v);
        f(v);
      }
    } else {
#pragma unroll 4
      for (int at = pieces.first + tid; at < pieces.last; at += kThreads) {
        float v[E];
        load16<T>(x + pieces.element(at), v);
        f(v);
      }
    }
  };
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int at = pieces.first + i * kThreads + tid;
      raw[i] = low_piece<T>();
      if (at < pieces.last) raw[i] = ld16raw<!TOP>(x + pieces.element(at));  // alternatives are read again
    }
  }
  float m = -INFINITY;
  each([&](const float* v) { m = fmaxf(m, max_of<E>(v)); });
  const float end = pieces.end();
  m = fmaxf(m, end);
  const float mine = m;
  m = wave_max(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  m = max_of<WAVES>(red[0]);
  const bool empty = m == -INFINITY;   // nothing is left (or NaN alone, which the sums keep)
  const float M = empty ? 0.f : m;
  float s = 0.f, w = 0.f;
  each([&](const float* v) { add_sums<E>(v, a.c, M, s, w); });
  add_sums<1>(&end, a.c, M, s, w);
  s = wave_sum(s);
  w = wave_sum(w);
  __syncthreads();
  if (lane == 0) {
    red[0][wave] = s;
    red[1][wave] = w;
  }
  __shared__ int count_s;
  __shared__ uint32_t group[64];
  if constexpr (TOP) {
    uint32_t of = score_key_asc(mine);
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) of = max(of, static_cast<uint32_t>(__shfl_xor(of, off)));
    static_assert(kThreads == 8 * 64, "64 groups of 8 lanes");
    if ((tid & 7) == 0) group[tid >> 3] = of;
    if (tid == 0) count_s = 0;
  }
  __syncthreads();
  s = w = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    s += red[0][i];
    w += red[1][i];
  }
  // x = -inf alone: every 2^t is 0, s = 0
  const float ls = __log2f(s);
  if (tid == 0) {
    const int64_t token = a.tokens[row];
    float lp = 0.f;
    if (token >= 0 && token < a.V) lp = s == 0.f ? -INFINITY : (to_f32(x[token]) - M) * a.inv_t - ls * kLn2;
    a.logp[row] = lp;
    a.entropy[row] = s == 0.f ? 0.f : (ls - w / s) * kLn2;
    if (a.stats) {
      a.stats[2 * row] = M;
      a.stats[2 * row + 1] = s;
    }
  }
  if constexpr (TOP) {
    __shared__ uint64_t list[kCandidates];
    auto put = [&](int place, uint64_t k) {
      const int e = static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
      a.top_tokens[row * a.K + place] = e;
      a.top[row * a.K + place] = s == 0.f ? -INFINITY : (to_f32(x[e]) - M) * a.inv_t - ls * kLn2;
    };
    int count = kCandidates + 1;
    if (s == s) {
      const float bound = score_of_key(kth_of_wave(group[lane], a.K));
      auto offer = [&](float v, int e) {
        if (v >= bound) {
          const int at = atomicAdd(&count_s, 1);
          if (at < kCandidates) list[at] = rank_key(v, e);
        }
      };
      auto offer_piece = [&](int at) {
        float v[E];
        load16<T>(x + pieces.element(at), v);
#pragma unroll
        for (int i = 0; i < E; ++i) offer(v[i], pieces.element(at) + i);
      };
      if (mine >= bound) {
        if (pieces.own >= 0) offer(end, pieces.own);
        if constexpr (NCH > 0) {
          uint32_t hits = 0;  // pieces that reach the bound: few
#pragma unroll
          for (int i = 0; i < NCH; ++i) {
            float v[E];
            unpack16<T>(raw[i], v);
            hits |= (max_of<E>(v) >= bound ? 1u : 0u) << i;
          }
          for (; hits != 0; hits &= hits - 1) {
            const int at = pieces.first + (__ffs(hits) - 1) * kThreads + tid;
            if (at < pieces.last) offer_piece(at);  // where the bound is -inf, what was never loaded reaches it
          }
        } else {
          for (int at = pieces.first + tid; at < pieces.last; at += kThreads) offer_piece(at);
        }
      }
      __syncthreads();
      count = count_s;
    }
    if (count <= 64) {  // the usual case: one wave ranks them, a candidate in each lane
      if (wave == 0) {
        const uint64_t k = lane < count ? list[lane] : 0;
        int above = 0;
        for (int j = 0; j < count; ++j) {
          const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(k >> 32), j);
          const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(k), j);
          above += ((static_cast<uint64_t>(hi) << 32) | lo) > k;
        }
        if (lane < count && above < a.K) put(above, k);
      }
    } else if (count <= kCandidates) {
      for (int i = tid; i < count; i += kThreads) {
        const uint64_t k = list[i];
        int above = 0;
        for (int j = 0; j < count; ++j) above += list[j] > k;
        if (above < a.K) put(above, k);
      }
    } else {
      uint64_t last = ~uint64_t(0);
      for (int place = 0; place < a.K; ++place) {
        uint64_t best = 0;
        for (int e = tid; e < a.V; e += kThreads) {
          const uint64_t k = rank_key(to_f32(x[e]), e);
          if (k < last && k > best) best = k;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
          const uint64_t o = shfl_xor64(best, off);
          best = o > best ? o : best;
        }
        __syncthreads();
        if (lane == 0) list[wave] = best;
        __syncthreads();
        best = list[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) best = list[i] > best ? list[i] : best;
        if (tid == 0) put(place, best);
        last = best;
      }
    }
  }
}

struct LogpGradArgs {
  const void* x;
  int64_t rs;
  const int64_t* tokens;
  const float *stats, *entropy;
  const float *g_logp, *g_entropy, *g_top;  // any may be null
  const int64_t* top_tokens;
  void* grad;  // [rows][V]
  int V, K, parts;
  float c, inv_t;
};

constexpr int kGradThreads = 256;
constexpr int kGradPieces = 8;  // of a thread

// Workgroup b takes part b % parts of row b / parts: 2048 pieces.
template <typename T, bool VEC>
__global__ __launch_bounds__(kGradThreads) void logp_grad_kernel(LogpGradArgs a) {
  constexpr int E = Vec<T>::N;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x - static_cast<int>(row) * a.parts, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.rs;
  T* out = static_cast<T*>(a.grad) + row * a.V;
  const Pieces<T> pieces(x, a.V);
  const float M = a.stats[2 * row], s = a.stats[2 * row + 1];
  const int64_t token = a.tokens[row];
  const bool given = token >= 0 && token < a.V;
  const float g_lp = a.g_logp && given ? a.g_logp[row] : 0.f;
  const float g_h = a.g_entropy ? a.g_entropy[row] : 0.f;
  float g_all = g_lp;
  if (a.g_top)
    for (int k = 0; k < a.K; ++k) g_all += a.g_top[row * a.K + k];
  const bool none = s == 0.f;  // a row of -inf alone: no gradient
  const float scale = none ? 0.f : -a.inv_t / s;
  const float A = scale * (g_all + (none ? 0.f : g_h * (a.entropy[row] - kLn2 * __log2f(s)))), B = scale * kLn2 * g_h;
  auto slope = [&](float v) {
    const float t = (v - M) * a.c;
    return __builtin_amdgcn_exp2f(t) * fmaf(B, fmaxf(t, kLowest), A);
  };
  // whole pieces; the ends of the row are the last part's
  const int begin = pieces.first + part * kGradThreads * kGradPieces;
  uint4 raw[kGradPieces];
#pragma unroll
  for (int i = 0; i < kGradPieces; ++i) {
    const int at = begin + i * kGradThreads + tid;
    if (at < pieces.last) raw[i] = ld16raw<true>(x + pieces.element(at));
  }
  auto value = [&](float v, int64_t e) { return slope(v) + (e == token && !none ? g_lp * a.inv_t : 0.f); };
  const int token_piece = given ? static_cast<int>((token + pieces.shift) / E) : -1;
#pragma unroll
  for (int i = 0; i < kGradPieces; ++i) {
    const int at = begin + i * kGradThreads + tid, e = pieces.element(at);
    if (at >= pieces.last) continue;
    float v[E];
    unpack16<T>(raw[i], v);
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = slope(v[k]);
    if (at == token_piece && !none) {
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] += e + k == token ? g_lp * a.inv_t : 0.f;
    }
    if constexpr (VEC) {
      store16<T, true>(out + e, v);
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) out[e + k] = from_f32<T>(v[k]);
    }
  }
  if (part == a.parts - 1 && pieces.own >= 0) out[pieces.own] = from_f32<T>(value(pieces.end(), pieces.own));
  if (a.g_top && !none) {  // the alternatives' own values once more, whole
    __syncthreads();
    for (int k = tid; k < a.K; k += kGradThreads) {
      const int64_t e = a.top_tokens[row * a.K + k];
      if (e < 0 || e >= a.V) continue;
      const int64_t at = (e + pieces.shift) / E;
      // whose is it: a whole piece's part, or the last part's end of the row
      const bool piece = at >= pieces.first && at < pieces.last;
      if (piece ? at < begin || at >= begin + kGradThreads * kGradPieces : part != a.parts - 1) continue;
      out[e] = from_f32<T>(value(to_f32(x[e]), e) + a.g_top[row * a.K + k] * a.inv_t);
    }
  }
}

// Positive, finite, and its inverse too.
bool good_temperature(float t) { return t > 0.f && t < INFINITY && kLog2e / t < INFINITY; }

// Workgroups of a launch: HIP counts its threads in 32 bits.
constexpr int64_t kMaxGroups = int64_t(1) << 22;

template <typename T>
T* at_row(T* p, int64_t at) { return p ? p + at : nullptr; }

template <typename T, bool TOP>
int launch_logp(LogpArgs a, int64_t rows, hipStream_t st) {
  constexpr int E = Vec<T>::N;
  const int64_t most = a.V / E;  // whole pieces
  for (int64_t row = 0; row < rows; row += kMaxGroups) {
    const int64_t here = rows - row < kMaxGroups ? rows - row : kMaxGroups;
    const dim3 grid(static_cast<unsigned>(here));
#define HYDRA_LOGP(N) logp_kernel<T, N, TOP><<<grid, kThreads, 0, st>>>(a)
    if (most <= 2 * kThreads) HYDRA_LOGP(2);
    else if (most <= 4 * kThreads) HYDRA_LOGP(4);
    else if (most <= 8 * kThreads) HYDRA_LOGP(8);
    else if (most <= 16 * kThreads) HYDRA_LOGP(16);
    else if (most <= 32 * kThreads) HYDRA_LOGP(32);
    else HYDRA_LOGP(0);
    const int rc = check_launch("token_logprobs");
    if (rc != HYDRA_OK) return rc;
    a.x = static_cast<const T*>(a.x) + here * a.rs;
    a.tokens += here;
    a.logp += here;
    a.entropy += here;
    a.stats = at_row(a.stats, 2 * here);
    a.top = at_row(a.top, here * a.K);
    a.top_tokens = at_row(a.top_tokens, here * a.K);
  }
#undef HYDRA_LOGP
  return HYDRA_OK;
}

template <typename T>
int launch_grad(LogpGradArgs a, int64_t rows, bool vec, hipStream_t st) {
  const int64_t most = kMaxGroups / a.parts;  // parts <= 2^17
  for (int64_t row = 0; row < rows; row += most) {
    const int64_t here = rows - row < most ? rows - row : most;
    const dim3 grid(static_cast<unsigned>(here * a.parts));
    if (vec) logp_grad_kernel<T, true><<<grid, kGradThreads, 0, st>>>(a);
    else logp_grad_kernel<T, false><<<grid, kGradThreads, 0, st>>>(a);
    const int rc = check_launch("token_logprobs_bwd");
    if (rc != HYDRA_OK) return rc;
    a.x = static_cast<const T*>(a.x) + here * a.rs;
    a.grad = static_cast<T*>(a.grad) + here * a.V;
    a.tokens += here;
    a.stats += 2 * here;
    a.entropy += here;
    a.g_logp = at_row(a.g_logp, here);
    a.g_entropy = at_row(a.g_entropy, here);
    a.g_top = at_row(a.g_top, here * a.K);
    a.top_tokens = at_row(a.top_tokens, here * a.K);
  }
  return HYDRA_OK;
}

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int hydra_token_logprobs(const void* logits, int64_t rows, int64_t vocab, int64_t logits_rs,
                                    const int64_t* tokens, float temperature, int64_t top_k, float* logprobs,
                                    float* entropy, float* stats, float* top_logprobs, int64_t* top_tokens, int dtype,
                                    void* stream) {
  HYDRA_REQUIRE(rows >= 0 && vocab >= 1, "token_logprobs: bad size");
  HYDRA_REQUIRE(vocab < (int64_t(1) << 30) && rows < (int64_t(1) << 31), "token_logprobs: too large");
  HYDRA_REQUIRE(logits_rs >= 0, "token_logprobs: negative row stride");
  HYDRA_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= vocab, "token_logprobs: need 0 <= top_k <= min(64, vocab)");
  HYDRA_REQUIRE(good_temperature(temperature), "token_logprobs: temperature must be positive and finite");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "token_logprobs: unknown dtype");
  if (rows == 0) return HYDRA_OK;
  HYDRA_REQUIRE(logits && tokens && logprobs && entropy && (top_k == 0 || (top_logprobs && top_tokens)),
                "token_logprobs: null pointer");
  HYDRA_REQUIRE(reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) == 0, "token_logprobs: misaligned logits");
  const LogpArgs a{logits, logits_rs, tokens, logprobs, entropy, stats, top_logprobs, top_tokens,
                   static_cast<int>(vocab), static_cast<int>(top_k), kLog2e / temperature, 1.f / temperature};
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return top_k > 0 ? launch_logp<T, true>(a, rows, st) : launch_logp<T, false>(a, rows, st);
  });
}

extern "C" int hydra_token_logprobs_bwd(const void* logits, int64_t rows, int64_t vocab, int64_t logits_rs,
                                        const int64_t* tokens, float temperature, int64_t top_k, const float* stats,
                                        const float* entropy, const int64_t* top_tokens, const float* g_logprobs,
                                        const float* g_entropy, const float* g_top, void* grad, int dtype,
                                        void* stream) {
  HYDRA_REQUIRE(rows >= 0 && vocab >= 1, "token_logprobs_bwd: bad size");
  HYDRA_REQUIRE(vocab < (int64_t(1) << 30) && rows < (int64_t(1) << 31), "token_logprobs_bwd: too large");
  HYDRA_REQUIRE(logits_rs >= 0, "token_logprobs_bwd: negative row stride");
  HYDRA_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= vocab,
                "token_logprobs_bwd: need 0 <= top_k <= min(64, vocab)");
  HYDRA_REQUIRE(good_temperature(temperature), "token_logprobs_bwd: temperature must be positive and finite");
  const int e = dtype_size(dtype);
  HYDRA_REQUIRE(e > 0, "token_logprobs_bwd: unknown dtype");
  if (rows == 0) return HYDRA_OK;
  HYDRA_REQUIRE(logits && tokens && stats && entropy && grad && (!g_top || top_tokens),
                "token_logprobs_bwd: null pointer");
  HYDRA_REQUIRE(reinterpret_cast<uintptr_t>(logits) % e == 0, "token_logprobs_bwd: misaligned logits");
  const int64_t most = vocab / (16 / e);  // whole pieces
  const int64_t parts = most == 0 ? 1 : (most + kGradThreads * kGradPieces - 1) / (kGradThreads * kGradPieces);
  const LogpGradArgs a{logits, logits_rs, tokens, stats, entropy, g_logprobs, g_entropy, g_top, top_tokens, grad,
                       static_cast<int>(vocab), static_cast<int>(top_k), static_cast<int>(parts),
                       kLog2e / temperature, 1.f / temperature};
  // A piece of the gradient is whole where the logits' is if rows start alike.
  const bool vec = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(grad)) % 16 == 0 &&
                   (rows <= 1 || (logits_rs - vocab) * e % 16 == 0);
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int { return launch_grad<T>(a, rows, vec, st); });
}
