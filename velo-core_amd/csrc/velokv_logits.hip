// velokv_logits.hip -- gfx950 kernels of the step from logits to tokens: log
// probabilities of given tokens, entropy, and the most probable tokens.
//
// A code object of its own (velokv_logits_gfx950.co), loaded beside the main one.
#include "velokv_device.h"

namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kLogitWaves = 4;
constexpr int kList = 512;       // candidates of a wave, ..
constexpr int kRoom = kList - 16;  // .. the values beside the vectors left out
constexpr int kStepValues = 32;  // values of a thread in a step

// =============================================================================
// Log probabilities of a row of logits x, in units of log 2: with c = scale log2(e) and
// m = max x,
//     e_v = (x_v - m) c,  Z = sum 2^e_v,  T = sum 2^e_v e_v,
//     log p_t = (x_t - m) scale - log2 Z ln 2,   entropy = (log2 Z - T / Z) ln 2,
// and the n_top largest x, ties to the lower index. One pass over the row: every
// thread keeps its own m, Z and T; a wave keeps a list of candidates for the largest
// values. A candidate is one 64-bit word, the value as an ordered key above the
// complement of its index, so that words differ and their order is the order wanted. In
// the first step a workgroup takes the n_top-th largest of the maxima of 32 groups of its
// lanes: at least n_top values reach it, and few more. Only those, and later values above
// it, are candidates. Where they may not fit the list (many equal values, rising ones) or
// fewer groups than n_top have a value (rows that a mask leaves little of, short rows), a
// wave takes its vectors one by one through LDS, the bound's equals up to n_top of them, and
// trims a full list (60 rows, one in eight masked to 1 % of 20000 fp32 values: 9.3 us with 5
// alternatives, 10.9 with 31 and 22 with 32).
//
// Bound: 1500 rows of 50001 fp16: 35 us, 150 MB at 4.3 TB/s (31 without alternatives), by the
// vector ALUs' work (ten instructions a value) beside the loads. 64 rows of 128000 fp16 with
// 20 alternatives: 14.5 us from the last-level cache and 15.0 from HBM, 8.6 without
// alternatives; every wave has one step, so its loads and its work do not overlap, and the
// join is a launch of its own (4.4 us). One row: launch and latency (32000 fp32: 8.5 us, 9.5
// from HBM). The exponent of base 2 is also the entropy's
// factor, which saves a product a value.
// =============================================================================
struct Sums { float m, z, t; };

// Sums taken from their maximum to the larger one m.
DEV Sums refer(const Sums& s, float m, float c) {
  const float e = s.m == m ? 0.0f : (s.m - m) * c, f = __builtin_amdgcn_exp2f(e);
  // (a factor of 0 may stand beside a product that is not finite)
  return Sums{m, f * s.z, f == 0.0f ? 0.0f : f * fmaf(s.z, e, s.t)};
}
// The wave's sums, in every lane.
DEV Sums wave_join(const Sums& s, float c) {
  const Sums a = refer(s, wave_max(s.m), c);
  return Sums{a.m, wave_sum(a.z), wave_sum(a.t)};
}

DEV uint64_t word_of(float x, int index) {
  return (uint64_t)order_key(x == x ? x : -kInf) << 32 | (uint32_t)~index;
}
DEV int word_index(uint64_t w) { return (int)~(uint32_t)w; }

// A bound that exactly k of a wave's words (N a lane, 0 = none) reach,
// found bit by bit from the first in which they differ; one that all reach where there are
// no more than k.
template <int N>
DEV uint64_t kth_word(const uint64_t (&x)[N], int k) {
  uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    most = max(most, (uint32_t)(x[i] >> 32));
    least = min(least, x[i] ? (uint32_t)(x[i] >> 32) : 0xFFFFFFFFu);
  }
  most = wave_max_u(most);
  least = ~wave_max_u(~least);
  // (an index has at most 28 bits)
  int bit = most > least ? 63 - __builtin_clz(most ^ least) : 27;
  uint64_t best = ((uint64_t)most << 32 | 0xF0000000u) >> bit >> 1 << 1 << bit;
  for (; bit >= 0; --bit) {
    const uint64_t t = best | 1ull << bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[i] >= t));
    if (count >= k) best = t;
    if (count == k) break;
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

// Leaves the k largest words of the list (n > k), which are those that reach `least`.
DEV int trim_list(uint64_t* list, int n, int k, uint64_t& least) {
  if (n <= WAVE) {  // a word a lane: its place is the number of larger ones
    const uint64_t x = lane_id() < n ? list[lane_id()] : 0;
    int place = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const uint64_t o = (uint64_t)(uint32_t)readlane_i((int)(x >> 32), j) << 32 | (uint32_t)readlane_i((int)x, j);
      place += o > x;
    }
    const int last = __builtin_ctzll(__builtin_amdgcn_ballot_w64(place == k - 1));
    least = (uint64_t)(uint32_t)readlane_i((int)(x >> 32), last) << 32 | (uint32_t)readlane_i((int)x, last);
    __builtin_amdgcn_wave_barrier();
    if (place < k) list[place] = x;
    return k;
  }
  uint64_t x[kList / WAVE];
#pragma unroll
  for (int i = 0; i < kList / WAVE; ++i) {
    const int at = i * WAVE + lane_id();
    x[i] = at < n ? list[at] : 0;
  }
  __builtin_amdgcn_wave_barrier();
  least = kth_word(x, k);
  return push_words(list, 0, x, least);
}

template <int DT>
DEV float logit(const LogprobParams& P, int row, int t) {
  const int64_t e = (int64_t)row * P.row_stride + t;
  return DT == DT_F32 ? reinterpret_cast<const float*>(P.logits)[e] : h2f(reinterpret_cast<const uint16_t*>(P.logits)[e]);
}
// The logit of given token i of a row; -infinity outside the vocabulary.
template <int DT>
DEV float token_logit(const LogprobParams& P, int row, int i) {
  const int t = P.tokens[(int64_t)row * P.n_tokens + i];
  return t >= 0 && t < P.vocab ? logit<DT>(P, row, t) : -kInf;
}

// The row's results from its sums and its k largest words, sorted; x0: the logit of the
// thread's first token.
template <int DT>
DEV void write_row(const LogprobParams& P, int row, const Sums& s, const uint64_t* top, float x0) {
  constexpr float kLn2 = 0.6931471805599453f;
  const bool none = s.m == -kInf && s.z == 0.0f;  // every logit is -infinity
  const float log_z = __builtin_log2f(s.z);
  const auto logprob = [&](float x) { return none ? -kInf : (x - s.m) * P.scale - log_z * kLn2; };
  const int tid = (int)threadIdx.x;
  for (int i = tid; i < P.n_tokens; i += (int)blockDim.x)
    P.token_logprobs[(int64_t)row * P.n_tokens + i] = logprob(i == tid ? x0 : token_logit<DT>(P, row, i));
  if (tid == 0 && P.entropy) P.entropy[row] = none ? 0.0f : (log_z - s.t / s.z) * kLn2;
  if (tid < P.n_top) {
    const int64_t at = (int64_t)row * P.n_top + tid;
    P.top_ids[at] = word_index(top[tid]);
    P.top_logprobs[at] = logprob(key_value((uint32_t)(top[tid] >> 32)));
  }
}

// Sorts words into top[0 .. k), largest first: each word's place is the number of larger
// ones. Eight lanes a word, which divide the others.
DEV void rank_words(const uint64_t* words, int n, int k, uint64_t* top) {
  const int sub = (int)threadIdx.x & 7;
  for (int i = (int)threadIdx.x >> 3; i < n; i += (int)blockDim.x >> 3) {
    const uint64_t x = words[i];
    int place = 0;
#pragma unroll 4
    for (int j = sub; j < n; j += 8) place += words[j] > x;
    place += (int)dpp_u<DPP_QUAD_XOR1>((uint32_t)place, 0);
    place += (int)dpp_u<DPP_QUAD_XOR2>((uint32_t)place, 0);
    place += (int)dpp_u<DPP_ROW_HALF_MIRROR>((uint32_t)place, 0);
    if (sub == 0 && place < k) top[place] = x;
  }
}

// One workgroup of W waves per (row, part). DT: the logits' type.
template <int DT, int W>
DEV void logprob_part(const LogprobParams& P) {
  constexpr int ESZ = DT == DT_F32 ? 4 : 2;
  constexpr int EPV = 16 / ESZ;             // values of a 16-byte vector
  constexpr int NV = kStepValues / EPV;     // vectors of a thread in a step
  constexpr int THREADS = W * WAVE;
  constexpr int GROUPS = 32 / W;            // groups of a wave's lanes
  __shared__ uint64_t lists[W][kList];
  __shared__ u32x4 staged[W][WAVE];
  __shared__ uint64_t words[W * kMaxTop];
  __shared__ uint64_t top[kMaxTop];
  __shared__ float sums[W][3];
  __shared__ __align__(16) float group_max[32];
  __shared__ int counts[W];
  const int tid = (int)threadIdx.x, lane = lane_id(), w = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int row = (int)(blockIdx.x / P.n_parts), part = (int)(blockIdx.x % P.n_parts);
  const int k = P.n_top;
  const float c = P.scale * kLog2e;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(P.logits) + (int64_t)row * P.row_stride * ESZ;
  // vectors are aligned: vector i holds values i EPV - off .. of the row. The values of
  // this part are [begin, end): the whole vectors [v_begin, v_end), and less than two
  // vectors of values beside them, one each for the first threads
  const int off = (int)(reinterpret_cast<uint64_t>(base) & 15) / ESZ;
  const int begin = part * P.part_len, end = min(P.vocab, begin + P.part_len);
  const int v_begin = (begin + off + EPV - 1) / EPV, v_end = max(v_begin, (end + off) / EPV);
  const int n_head = min(end, v_begin * EPV - off) - begin;
  const int extra = tid < n_head ? begin + tid : v_end * EPV - off + tid - n_head;
  const bool has_extra = extra < end && tid < 2 * EPV;
  float x_extra = -kInf;
  if (has_extra)
    x_extra = DT == DT_F32 ? reinterpret_cast<const float*>(base)[extra] : h2f(reinterpret_cast<const uint16_t*>(base)[extra]);

  // (no load sits in a branch: threads past the last vector load it again, and step()
  // takes -infinity in its place)
  const auto load = [&](u32x4(&r)[NV], int v0) {
    if (v_end == v_begin) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = min(v0 + i * THREADS + tid, v_end - 1);
      r[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(base + ((int64_t)v * EPV - off) * ESZ));
    }
  };
  const auto value = [](const u32x4& r, int e) {
    return DT == DT_F32 ? bitcast<float>(r[e]) : e % 2 ? half_hi(r[e / 2]) : half_lo(r[e / 2]);
  };

  const float x0 = P.n_parts == 1 && tid < P.n_tokens ? token_logit<DT>(P, row, tid) : -kInf;
  Sums s{-kInf, 0.0f, 0.0f};
  float thr_x = -kInf;   // candidates of later steps are larger
  int n = 0;             // candidates in the list
  uint64_t* list = lists[w];
  // Vector rv of every lane, 64 values at a time in the order of their indices: those above
  // thr_x and the first `equals` that equal it. A full list is trimmed and gives a higher
  // bound (values that equal it come later than those listed, and lose to them).
  const auto take_vector = [&](const u32x4& rv, int v, int& equals) {
    __builtin_amdgcn_wave_barrier();
    staged[w][lane] = rv;
    __builtin_amdgcn_wave_barrier();
    const int at = (v - lane) * EPV - off, limit = v_end * EPV - off;
    constexpr int EB = 4;  // read together
#pragma unroll 1
    for (int e0 = 0; e0 < EPV; e0 += EB) {
      if (n > kRoom - EB * WAVE) {
        uint64_t least;
        n = trim_list(list, n, k, least);
        thr_x = fmaxf(thr_x, key_value((uint32_t)(least >> 32)));
        equals = 0;
      }
      float xs[EB];
#pragma unroll
      for (int e = 0; e < EB; ++e)
        xs[e] = DT == DT_F32 ? reinterpret_cast<const float*>(staged[w])[(e0 + e) * WAVE + lane]
                             : h2f(reinterpret_cast<const uint16_t*>(staged[w])[(e0 + e) * WAVE + lane]);
#pragma unroll
      for (int e = 0; e < EB; ++e) {
        const int index = at + (e0 + e) * WAVE + lane;
        const bool more = index < limit && xs[e] > thr_x;
        uint64_t mask = __builtin_amdgcn_ballot_w64(more);
        const uint64_t below = (1ull << lane) - 1;
        bool in = more;
        if (equals > 0) {
          const bool equal = index < limit && (thr_x == -kInf ? !more : xs[e] == thr_x);
          const uint64_t em = __builtin_amdgcn_ballot_w64(equal);
          in = more || (equal && __builtin_popcountll(em & below) < equals);
          mask = __builtin_amdgcn_ballot_w64(in);
          equals -= __builtin_popcountll(em);
        }
        if (mask == 0) continue;
        if (in) list[n + __builtin_popcountll(mask & below)] = word_of(xs[e], index);
        n += __builtin_popcountll(mask);
      }
    }
  };
  const auto step = [&](u32x4(&r)[NV], int v0, bool first) {
    if (v0 + NV * THREADS > v_end) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = v0 + i * THREADS + tid < v_end;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[i][j] = in ? r[i][j] : DT == DT_F32 ? 0xFF800000u : 0xFC00FC00u;
      }
    }
    float x[NV][EPV], vm[NV], mv = -kInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < EPV; ++e) x[i][e] = value(r[i], e);
      vm[i] = fmaxf(x[i][0], x[i][1]);
#pragma unroll
      for (int e = 2; e < EPV; ++e) vm[i] = fmaxf(vm[i], x[i][e]);
      mv = fmaxf(mv, vm[i]);
    }
    const float m = first ? fmaxf(mv, x_extra) : mv;
    if (k > 0) {
      if (first) {
        // the maxima of 32 groups of lanes (the vectors' alone: values
        // of later steps may come before the row's last ones, which are among the extra)
        float gm = fmaxf(mv, dpp<DPP_QUAD_XOR1>(mv));
        gm = fmaxf(gm, dpp<DPP_QUAD_XOR2>(gm));
        gm = fmaxf(gm, dpp<DPP_ROW_HALF_MIRROR>(gm));
        if constexpr (GROUPS == 2) {
          gm = fmaxf(gm, dpp<DPP_ROW_MIRROR>(gm));
          gm = fmaxf(gm, shfl_xor(gm, 16));
        }
        if (lane % (WAVE / GROUPS) == 0) group_max[w * GROUPS + lane / (WAVE / GROUPS)] = gm;
        __syncthreads();
        const float mine = group_max[lane & 31];
        if (k > 1) {  // the largest that k of them reach
          int reach = 0;  // lanes 32 apart hold the same group and count half of them each
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 o = reinterpret_cast<const float4*>(group_max)[4 * (lane >> 5) + j];
            reach += (o.x >= mine) + (o.y >= mine) + (o.z >= mine) + (o.w >= mine);
          }
          reach += __float_as_int(xor32(__int_as_float(reach)));
          thr_x = wave_max(reach >= k ? mine : -kInf);
        } else {
          thr_x = wave_max(mine);
        }
      }
      // candidates: at least thr_x in the first step, above it later
      if (__builtin_amdgcn_ballot_w64(first || mv > thr_x) != 0) {
        // what the list may have to take, by vectors. Where that is too much (a mask's equal
        // values, rising ones) or no bound is known (fewer groups than n_top with a value),
        // the vectors are taken one by one
        uint64_t hit[NV];
        int count = n;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          hit[i] = __builtin_amdgcn_ballot_w64(first ? vm[i] >= thr_x : vm[i] > thr_x);
          count += EPV * __builtin_popcountll(hit[i]);
        }
        if (count <= kRoom && !(first && thr_x == -kInf)) {
          const uint64_t below = (1ull << lane) - 1;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            if (hit[i] == 0) continue;
#pragma unroll
            for (int e = 0; e < EPV; ++e) {
              const bool in = first ? x[i][e] >= thr_x : x[i][e] > thr_x;
              const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
              if (mask == 0) continue;
              if (in) list[n + __builtin_popcountll(mask & below)] = word_of(x[i][e], (v0 + i * THREADS + tid) * EPV - off + e);
              n += __builtin_popcountll(mask);
            }
          }
        } else {
          int equals = first ? k : 0;
#pragma unroll 1
          for (int i = 0; i < NV && v0 + i * THREADS + w * WAVE < v_end; ++i) {
            u32x4 rv = r[0];
#pragma unroll
            for (int j = 1; j < NV; ++j) {
              const u32x4 o = r[j];
#pragma unroll
              for (int d = 0; d < 4; ++d) rv[d] = i == j ? o[d] : rv[d];
            }
            take_vector(rv, v0 + i * THREADS + tid, equals);
          }
          if (n > kRoom / 2) {
            uint64_t least;
            n = trim_list(list, n, k, least);
            thr_x = fmaxf(thr_x, key_value((uint32_t)(least >> 32)));
          }
        }
      }
    }
    if (m > s.m) s = refer(s, m, c);
    const float ref = s.m == -kInf ? 0.0f : s.m;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const float y = (x[i][e] - ref) * c, p = __builtin_amdgcn_exp2f(y);
        s.z += p;
        s.t = fmaf(p, fmaxf(y, -3e38f), s.t);  // (p is 0 where y is -infinity)
      }
    if (first) {
      const float y = (x_extra - ref) * c, p = __builtin_amdgcn_exp2f(y);
      s.z += p;
      s.t = fmaf(p, fmaxf(y, -3e38f), s.t);
    }
  };

  u32x4 a[NV], b[NV];
  constexpr int STEP = NV * THREADS;
  load(a, v_begin);
  load(b, v_begin + STEP);
  step(a, v_begin, true);
  for (int v = v_begin + STEP; v < v_end; v += 2 * STEP) {
    load(a, v + STEP);
    step(b, v, false);
    if (v + STEP >= v_end) break;
    load(b, v + 2 * STEP);
    step(a, v + STEP, false);
  }

  if (k > 0 && w == 0) {  // the values beside the vectors, which have their threads in wave 0
    static_assert(2 * EPV <= kList - kRoom && 2 * EPV <= WAVE, "room for them");
    const bool in = has_extra && !(x_extra < thr_x);
    const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
    if (in) list[n + __builtin_popcountll(mask & ((1ull << lane) - 1))] = word_of(x_extra, extra);
    n += __builtin_popcountll(mask);
  }
  s = wave_join(s, c);
  if (lane == 0) { sums[w][0] = s.m; sums[w][1] = s.z; sums[w][2] = s.t; }
  if (k > 0) {
    uint64_t least;
    if (n > kMaxTop) n = trim_list(list, n, k, least);
    if (lane == 0) counts[w] = n;
  }
  if (tid < k) top[tid] = 0;
  __syncthreads();
  {
    float m = sums[0][0];
#pragma unroll
    for (int i = 1; i < W; ++i) m = fmaxf(m, sums[i][0]);
    s = Sums{m, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const Sums o = refer(Sums{sums[i][0], sums[i][1], sums[i][2]}, m, c);
      s.z += o.z;
      s.t += o.t;
    }
  }
  if (k > 0) {
    int at = 0, total = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) { at += i < w ? counts[i] : 0; total += counts[i]; }
    if (lane < n) words[at + lane] = list[lane];
    __syncthreads();
    rank_words(words, total, k, top);
    __syncthreads();
  }
  if (P.n_parts == 1) {
    write_row<DT>(P, row, s, top, x0);
    return;
  }
  const int64_t pr = (int64_t)row * P.n_parts + part;
  if (tid == 0) reinterpret_cast<float4*>(P.part_sums)[pr] = make_float4(s.m, s.z, s.t, 0.0f);
  if (tid < k) P.part_top[pr * k + tid] = top[tid];
}

// The parts of a row.
template <int DT>
DEV void logprob_join(const LogprobParams& P) {
  __shared__ uint64_t words[kMaxLogitParts * kMaxTop];
  __shared__ uint64_t top[kMaxTop];
  __shared__ int count;
  const int tid = (int)threadIdx.x, lane = lane_id(), row = (int)blockIdx.x, k = P.n_top, n = P.n_parts * k;
  const float c = P.scale * kLog2e;
  // every wave joins the sums by itself, one part a lane; what the row needs of memory is
  // asked for at once
  static_assert(kMaxLogitParts <= WAVE, "a part a lane");
  constexpr int NT = kMaxLogitParts * kMaxTop / (WAVE * kLogitWaves);  // words of a thread
  const bool in_part = lane < P.n_parts;
  const float4 ps = reinterpret_cast<const float4*>(P.part_sums)[(int64_t)row * P.n_parts + (in_part ? lane : 0)];
  const uint64_t* in = P.part_top + (int64_t)row * n;
  // the need-th largest of the parts' at_least-th words is reached by need x at_least >= k
  // words, of the parts' k each; some half more than k reach it
  const int at_least = min(k, (5 * k + 4 * P.n_parts - 1) / (4 * P.n_parts)), need = (k + at_least - 1) / max(at_least, 1);
  uint32_t nth = 0;
  uint64_t word[NT] = {};  // 0: no word
  if (k > 0) {
#pragma unroll
    for (int i = 0; i < NT; ++i) word[i] = in[min(tid + i * WAVE * kLogitWaves, n - 1)];
    nth = (uint32_t)(in[(in_part ? lane : 0) * k + at_least - 1] >> 32);
    if (tid == 0) count = 0;
    if (tid < k) top[tid] = 0;
  }
  const float x0 = tid < P.n_tokens ? token_logit<DT>(P, row, tid) : -kInf;
  const Sums s = wave_join(in_part ? Sums{ps.x, ps.y, ps.z} : Sums{-kInf, 0.0f, 0.0f}, c);
  if (k > 0) {
    int reach = 0;
    for (int j = 0; j < P.n_parts; j += 8)
#pragma unroll
      for (int e = 0; e < 8; ++e) reach += j + e < P.n_parts && (uint32_t)readlane_i((int)nth, j + e) >= nth;
    const uint64_t least = max(1ull, (uint64_t)wave_max_u(in_part && reach >= need ? nth : 0u) << 32);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const bool keep = tid + i * WAVE * kLogitWaves < n && word[i] >= least;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(keep);
      if (mask == 0) continue;
      int at = 0;
      if (lane == 0) at = atomicAdd(&count, __builtin_popcountll(mask));
      at = __builtin_amdgcn_readfirstlane(at);
      if (keep) words[at + __builtin_popcountll(mask & ((1ull << lane) - 1))] = word[i];
    }
    __syncthreads();
    rank_words(words, count, k, top);
    __syncthreads();
  }
  write_row<DT>(P, row, s, top, x0);
}

}  // namespace

#define VK_FOUR_WAVES __attribute__((amdgpu_waves_per_eu(4)))
#define VK_LOGITS(DT)                                                                                                             \
  extern "C" __global__ void __launch_bounds__(WAVE* kLogitWaves) VK_FOUR_WAVES vk_logprob_part_q##DT(const LogprobParams P) {       \
    logprob_part<DT, kLogitWaves>(P);                                                                                               \
  }                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(1024) vk_logprob_row_q##DT(const LogprobParams P) { logprob_part<DT, 16>(P); }        \
  extern "C" __global__ void __launch_bounds__(WAVE* kLogitWaves) vk_logprob_join_q##DT(const LogprobParams P) { logprob_join<DT>(P); }
VK_LOGITS(0) VK_LOGITS(1)
