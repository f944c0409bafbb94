// velokv_logits.hip -- gfx950 kernels of the step from logits to tokens: log
// probabilities of given tokens, entropy, and the most probable tokens.
//
// A code object of its own (velokv_logits_gfx950.co), loaded beside the main one.
#include "velokv_device.h"

namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kLogitWaves = 4;
constexpr int kLogitThreads = WAVE * kLogitWaves;
constexpr int kList = 512;  // candidates of a wave

// =============================================================================
// Log probabilities of a row x (logits times scale): with M = max x,
//     Z = sum e^(x - M),  T = sum e^(x - M) (x - M),
//     log p_t = (x_t - M) - log Z,   entropy = log Z - T / Z,
// and the n_top largest x, ties to the lower index. One pass over the row: every
// thread keeps its own running M, Z and T; a wave keeps a list of candidates for the
// largest values. A candidate is one 64-bit word, the value as an ordered key above
// the complement of its index, so that words differ and their order is the order
// wanted. thr is a word that at least n_top of the wave's words reach: only larger
// ones are added, and after the first vectors of a row few are.
// =============================================================================
struct Sums { float m, z, t; };

// a and b joined; c = scale * log2(e).
DEV Sums join(const Sums& a, const Sums& b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -kInf) return Sums{m, a.z + b.z, a.t + b.t};  // sums are 0, or NaN
  const float fa = __builtin_amdgcn_exp2f((a.m - m) * c), fb = __builtin_amdgcn_exp2f((b.m - m) * c);
  Sums r{m, fa * a.z + fb * b.z, 0.0f};
  // (a factor of 0 stands beside sums whose product with the distance may overflow)
  if (fa != 0.0f) r.t += fa * (a.t + a.z * (a.m - m));
  if (fb != 0.0f) r.t += fb * (b.t + b.z * (b.m - m));
  return r;
}
DEV Sums wave_join(Sums a, float c) {
#pragma unroll
  for (int m = 1; m < WAVE; m *= 2) a = join(a, Sums{shfl_xor(a.m, m), shfl_xor(a.z, m), shfl_xor(a.t, m)}, c);
  return a;
}

DEV uint64_t word_of(float x, int index) {
  return (uint64_t)order_key(x == x ? x : -kInf) << 32 | (uint32_t)~index;
}
DEV int word_index(uint64_t w) { return (int)~(uint32_t)w; }

// The k-th largest of a wave's words (N a lane, 0 = none): the largest word that k of
// them reach, found bit by bit; 0 where there are fewer than k.
template <int N>
DEV uint64_t kth_word(const uint64_t (&x)[N], int k) {
  uint64_t best = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t t = best | 1ull << bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[i] >= t));
    if (count >= k) best = t;
  }
  return best;
}

// Adds the lanes' words that reach `least` to the list; returns its new length.
template <int N>
DEV int push_words(uint64_t* list, int n, const uint64_t (&x)[N], uint64_t least) {
  const uint64_t below = (1ull << lane_id()) - 1;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = x[i] >= least && x[i] != 0;
    const uint64_t m = __builtin_amdgcn_ballot_w64(in);
    if (in) list[n + __builtin_popcountll(m & below)] = x[i];
    n += __builtin_popcountll(m);
  }
  return n;
}

// Leaves the k largest words of the list (n > k).
DEV int trim_list(uint64_t* list, int n, int k) {
  uint64_t x[kList / WAVE];
#pragma unroll
  for (int i = 0; i < kList / WAVE; ++i) {
    const int at = i * WAVE + lane_id();
    x[i] = at < n ? list[at] : 0;
  }
  __builtin_amdgcn_wave_barrier();
  const uint64_t least = kth_word(x, k);
  return push_words(list, 0, x, least);
}

// The row's results from its sums and its k largest words, sorted.
template <int DT>
DEV void write_row(const LogprobParams& P, int row, const Sums& s, const uint64_t* top) {
  const float log_z = logf(s.z);
  const auto logprob = [&](float x) { return s.m == -kInf && s.z == 0.0f ? -kInf : (x - s.m) * P.scale - log_z; };
  const int tid = (int)threadIdx.x;
  for (int i = tid; i < P.n_tokens; i += kLogitThreads) {
    const int64_t at = (int64_t)row * P.n_tokens + i;
    const int t = P.tokens[at];
    float x = -kInf;
    if (t >= 0 && t < P.vocab) {
      const int64_t e = (int64_t)row * P.row_stride + t;
      x = DT == DT_F32 ? reinterpret_cast<const float*>(P.logits)[e] : h2f(reinterpret_cast<const uint16_t*>(P.logits)[e]);
    }
    P.token_logprobs[at] = logprob(x);
  }
  if (tid == 0 && P.entropy) P.entropy[row] = s.m == -kInf && s.z == 0.0f ? 0.0f : log_z - s.t / s.z * P.scale;
  if (tid < P.n_top) {
    const int64_t at = (int64_t)row * P.n_top + tid;
    P.top_ids[at] = word_index(top[tid]);
    P.top_logprobs[at] = logprob(key_value((uint32_t)(top[tid] >> 32)));
  }
}

// Sorts words into top[0 .. k), largest first: each word's place is the number of larger ones.
DEV void rank_words(const uint64_t* words, int n, int k, uint64_t* top) {
  for (int i = (int)threadIdx.x; i < n; i += kLogitThreads) {
    const uint64_t x = words[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += words[j] > x;
    if (place < k) top[place] = x;
  }
}

template <int DT>
DEV void logprob_part(const LogprobParams& P) {
  constexpr int ESZ = DT == DT_F32 ? 4 : 2;
  constexpr int EPV = 16 / ESZ;     // values of a 16-byte vector
  constexpr int NV = 32 / EPV;      // vectors of a thread in a step
  __shared__ uint64_t lists[kLogitWaves][kList];
  __shared__ uint64_t words[kLogitWaves * kMaxTop];
  __shared__ uint64_t top[kMaxTop];
  __shared__ float sums[kLogitWaves][3];
  __shared__ int counts[kLogitWaves];
  const int tid = (int)threadIdx.x, lane = lane_id(), w = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int row = (int)(blockIdx.x / P.n_parts), part = (int)(blockIdx.x % P.n_parts);
  const int k = P.n_top;
  const float c = P.scale * kLog2e;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(P.logits) + (int64_t)row * P.row_stride * ESZ;
  // vectors are aligned: vector i holds values i EPV - off .. of the row; the values of
  // this part are [begin, end)
  const int off = (int)(reinterpret_cast<uint64_t>(base) & 15) / ESZ;
  const int begin = part * P.part_len, end = min(P.vocab, begin + P.part_len);
  const int v_begin = (begin + off) / EPV, v_end = (end + off + EPV - 1) / EPV;

  const auto load = [&](u32x4(&r)[NV], int v0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = v0 + i * kLogitThreads + tid, at = v * EPV - off;
      if (at >= begin && at + EPV <= end) {
        r[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(base + (int64_t)at * ESZ));
      } else {  // the row's ends
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
          uint32_t b = DT == DT_F32 ? 0xFF800000u : 0xFC00u;  // -infinity
          if (v < v_end && at + e >= begin && at + e < end)
            b = DT == DT_F32 ? reinterpret_cast<const uint32_t*>(base)[at + e] : reinterpret_cast<const uint16_t*>(base)[at + e];
          if constexpr (DT == DT_F32) r[i][e] = b;
          else r[i][e / 2] = e % 2 ? r[i][e / 2] | b << 16 : b;
        }
      }
    }
  };

  Sums s{-kInf, 0.0f, 0.0f};
  uint64_t thr = 0;
  float thr_x = 0.0f;
  int n = 0;
  uint64_t* list = lists[w];
  const auto step = [&](const u32x4(&r)[NV], int v0) {
    float x[NV][EPV], vmax[NV], m = -kInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      vmax[i] = -kInf;
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        x[i][e] = DT == DT_F32 ? bitcast<float>(r[i][e]) : e % 2 ? half_hi(r[i][e / 2]) : half_lo(r[i][e / 2]);
        vmax[i] = fmaxf(vmax[i], x[i][e]);
      }
      m = fmaxf(m, vmax[i]);
    }
    if (m > s.m) {
      const float f = __builtin_amdgcn_exp2f((s.m - m) * c);
      s.t = f == 0.0f ? 0.0f : f * (s.t + s.z * (s.m - m));
      s.z *= f;
      s.m = m;
    }
    const float at = s.m == -kInf ? 0.0f : s.m;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const float d = x[i][e] - at, p = __builtin_amdgcn_exp2f(d * c);
        s.z += p;
        s.t += p == 0.0f ? 0.0f : p * d;
      }
    if (k == 0) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (__builtin_amdgcn_ballot_w64(thr == 0 || vmax[i] > thr_x) == 0) continue;
      uint64_t word[EPV], most[1] = {0};
      const int first = (v0 + i * kLogitThreads + tid) * EPV - off;
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        word[e] = first + e >= begin && first + e < end ? word_of(x[i][e], first + e) : 0;
        most[0] = word[e] > most[0] ? word[e] : most[0];
      }
      // fewer than k lanes hold a larger word than the k-th largest of the lanes' largest:
      // at most (kMaxTop - 1) EPV + 1 words reach it
      const uint64_t kth = kth_word(most, k);
      if (n > kList - kMaxTop * EPV) n = trim_list(list, n, k);
      n = push_words(list, n, word, max(kth, thr));
      if (kth > thr) {
        thr = kth;
        thr_x = key_value((uint32_t)(thr >> 32));
      }
    }
  };

  u32x4 a[NV], b[NV];
  constexpr int STEP = NV * kLogitThreads;
  load(a, v_begin);
  for (int v = v_begin; v < v_end; v += 2 * STEP) {
    load(b, v + STEP);
    step(a, v);
    if (v + STEP >= v_end) break;
    load(a, v + 2 * STEP);
    step(b, v + STEP);
  }

  s = wave_join(s, c);
  if (lane == 0) { sums[w][0] = s.m; sums[w][1] = s.z; sums[w][2] = s.t; }
  if (k > 0) {
    if (n > kMaxTop) n = trim_list(list, n, k);
    if (lane == 0) counts[w] = n;
  }
  __syncthreads();
  s = Sums{sums[0][0], sums[0][1], sums[0][2]};
  for (int i = 1; i < kLogitWaves; ++i) s = join(s, Sums{sums[i][0], sums[i][1], sums[i][2]}, c);
  if (k > 0) {
    int at = 0, total = 0;
    for (int i = 0; i < kLogitWaves; ++i) { at += i < w ? counts[i] : 0; total += counts[i]; }
    if (lane < n) words[at + lane] = list[lane];
    if (tid < k) top[tid] = 0;
    __syncthreads();
    rank_words(words, total, k, top);
    __syncthreads();
  }
  if (P.n_parts == 1) {
    write_row<DT>(P, row, s, top);
    return;
  }
  const int64_t pr = (int64_t)row * P.n_parts + part;
  if (tid == 0) reinterpret_cast<float4*>(P.part_sums)[pr] = make_float4(s.m, s.z, s.t, 0.0f);
  if (tid < k) P.part_top[pr * k + tid] = top[tid];
}

// The parts of a row. A word can be among the k largest only if it reaches the largest
// of the parts' k-th words.
template <int DT>
DEV void logprob_join(const LogprobParams& P) {
  __shared__ uint64_t words[kMaxLogitParts * kMaxTop];
  __shared__ uint64_t top[kMaxTop];
  __shared__ int count;
  const int tid = (int)threadIdx.x, row = (int)blockIdx.x, k = P.n_top, n = P.n_parts * k;
  const float c = P.scale * kLog2e;
  const float4* parts = reinterpret_cast<const float4*>(P.part_sums) + (int64_t)row * P.n_parts;
  Sums s{parts[0].x, parts[0].y, parts[0].z};
  for (int i = 1; i < P.n_parts; ++i) s = join(s, Sums{parts[i].x, parts[i].y, parts[i].z}, c);
  if (k > 0) {
    const uint64_t* in = P.part_top + (int64_t)row * n;
    uint64_t least = 1;  // 0: no word
    for (int i = 0; i < P.n_parts; ++i) least = max(least, in[i * k + k - 1]);
    if (tid == 0) count = 0;
    if (tid < k) top[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kLogitThreads) {
      const uint64_t x = in[i];
      if (x >= least) words[atomicAdd(&count, 1)] = x;
    }
    __syncthreads();
    rank_words(words, count, k, top);
    __syncthreads();
  }
  write_row<DT>(P, row, s, top);
}

}  // namespace

#define VK_LOGITS(DT)                                                                                                  \
  extern "C" __global__ void __launch_bounds__(kLogitThreads) vk_logprob_part_q##DT(const LogprobParams P) { logprob_part<DT>(P); } \
  extern "C" __global__ void __launch_bounds__(kLogitThreads) vk_logprob_join_q##DT(const LogprobParams P) { logprob_join<DT>(P); }
VK_LOGITS(0) VK_LOGITS(1)
