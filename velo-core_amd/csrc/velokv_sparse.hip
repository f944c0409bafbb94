// velokv_sparse.hip -- gfx950 kernels of sparse decode: the key index beside a
// pool, the choice of pages by it, and attention over the chosen pages.
//
// A code object of its own (velokv_sparse_gfx950.co), loaded beside the main one.
#include "velokv_device.h"

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef short short2v __attribute__((ext_vector_type(2)));

namespace {

constexpr float kInf = __builtin_huge_valf();

DEV int table_row(const int32_t* seq_rows, int s, int bt_rows) {
  const int row = seq_rows ? seq_rows[s] : s;
  return bt_rows > 0 ? min(max(row, 0), bt_rows - 1) : row;
}
DEV bool finite(float x) { return fabsf(x) < kInf; }
// 127 / top, 0 where that is not finite (top 0, denormal, infinite or NaN).
DEV float code_scale(float top) {
  const float inv = 127.0f / top;
  return finite(inv) ? inv : 0.0f;
}
DEV int to_code(float x, float inv) { return (int)fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f); }

// =============================================================================
// Key index: for a page and KV head lo[d] = min_t k[t][d], hi[d] = max_t k[t][d]
// over the page's tokens below the context's end, as int8 codes rint(x 127 / top)
// with one fp32 scale top / 127, top = max_d max(|lo|, |hi|). One wave per (page,
// KV head): lanes take 16-byte chunks of the K tiles, so each holds the bounds of a
// fixed set of dims and the tokens' lanes are joined by lane exchanges at the end.
// A code is the nearest, so a bound may lie up to half a step (top / 254) inside the
// keys' range. A page with a key that is not finite has the scale infinity (it is chosen
// before any other).
// Bound: the chain of table, keys and codes. The newest pages of 64 sequences x 8 heads
// (fp16): 3.4 us; 4 int8 prompts of 1500-2500 tokens x 8 heads: 7.6 us for 9 MB. The
// loads of a tile are all in flight at once.
// =============================================================================
// Exchanges x's lanes with bit M set and y's without: afterwards a lane without it
// holds both halves of x, one with it both of y.
template <int M>
DEV void swap_lanes(uint32_t& x, uint32_t& y) {
  const auto r = M == 32 ? __builtin_amdgcn_permlane32_swap(x, y, false, false) : __builtin_amdgcn_permlane16_swap(x, y, false, false);
  x = r[0];
  y = r[1];
}
template <int M>
DEV void swap_lanes(float& x, float& y) {
  uint32_t a = bitcast<uint32_t>(x), b = bitcast<uint32_t>(y);
  swap_lanes<M>(a, b);
  x = bitcast<float>(a);
  y = bitcast<float>(b);
}
// Bounds of dims as signed integers, one (fp32) or two (PK: 16 bits each) a word.
// Integers take one instruction a comparison; a float minimum of a value from another
// lane takes two.
template <bool PK>
DEV uint32_t word_min(uint32_t a, uint32_t b) {
  if constexpr (PK) return bitcast<uint32_t>(__builtin_elementwise_min(bitcast<short2v>(a), bitcast<short2v>(b)));
  else return (uint32_t)min((int)a, (int)b);
}
template <bool PK>
DEV uint32_t word_max(uint32_t a, uint32_t b) {
  if constexpr (PK) return bitcast<uint32_t>(__builtin_elementwise_max(bitcast<short2v>(a), bitcast<short2v>(b)));
  else return (uint32_t)max((int)a, (int)b);
}
// A float's bits as an integer of the same order, NaN beyond infinity, and back (the map
// is its own inverse).
DEV uint32_t ordered_f32(uint32_t x) { return x ^ (uint32_t)((int)x >> 31) >> 1; }
DEV uint32_t ordered_f16x2(uint32_t x) {
  const short2v s = bitcast<short2v>(x);
  return x ^ (bitcast<uint32_t>(s >> (short)15) & 0x7FFF7FFFu);
}
// Joins lanes l and l ^ M: lanes with bit M clear are left the first half of the N
// words, the others the second, in [0, N / 2).
template <bool PK, int N, int M>
DEV void fold_lanes(uint32_t* lo, uint32_t* hi) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    swap_lanes<M>(lo[i], lo[i + N / 2]);
    swap_lanes<M>(hi[i], hi[i + N / 2]);
    lo[i] = word_min<PK>(lo[i], lo[i + N / 2]);
    hi[i] = word_max<PK>(hi[i], hi[i + N / 2]);
  }
}
// Over the lanes of a row of 16 that are equal mod LPT.
template <bool PK, int CTRL, int N>
DEV void join_turned(uint32_t* lo, uint32_t* hi) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    lo[i] = word_min<PK>(lo[i], dpp_u<CTRL>(lo[i], lo[i]));
    hi[i] = word_max<PK>(hi[i], dpp_u<CTRL>(hi[i], hi[i]));
  }
}
template <bool PK, int LPT, int N>
DEV void join_row(uint32_t* lo, uint32_t* hi) {
  if constexpr (LPT <= 8) join_turned<PK, DPP_ROW_ROR8, N>(lo, hi);
  if constexpr (LPT <= 4) join_turned<PK, DPP_ROW_ROR4, N>(lo, hi);
  if constexpr (LPT <= 2) join_turned<PK, DPP_ROW_ROR2, N>(lo, hi);
}

constexpr int kUpdateThreads = 256;

template <int KV, int T>
DEV void index_update(const IndexUpdateParams& P) {
  constexpr int ESZ = Esz<KV>::v;
  constexpr bool I8 = ESZ == 1, BLK = KV == KV_I8_BLK, REF = KV == KV_I8_REF;
  constexpr bool PK = KV == KV_F16 || BLK;           // two dims a word
  constexpr int EPC = 16 / ESZ;                      // dims of a 16-byte chunk
  constexpr int LPT = I8 ? T / 32 : T / EPC;         // lanes that hold one token's chunks of a load
  constexpr int NI = 16 * T * ESZ / 1024;            // loads of 64 chunks per tile
  constexpr int NS = (I8 && T == 128) ? 2 : 1;       // sets of dims a lane holds
  constexpr int NW = NS * EPC / (PK ? 2 : 1);        // words a lane holds
  constexpr bool R16 = LPT <= 16, R32 = !(I8 && T == 64);  // lanes 16 (32) apart hold the same dims
  constexpr int N1 = R32 ? NW / 2 : NW, NF = R16 ? N1 / 2 : N1;  // words left after each exchange
  constexpr int NO = NF * (PK ? 2 : 1);              // dims a lane is left with, side by side
  const int lane = lane_id();
  const int wg = P.wg0 + (int)blockIdx.x, s = wg / P.seq_wgs;
  const int unit = (wg - s * P.seq_wgs) * (kUpdateThreads / WAVE) + __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int nth = unit / P.n_kv_heads, kvh = unit - nth * P.n_kv_heads;
  if (nth >= P.max_pages) return;
  const int ctx = max(0, min(P.context_lens[s], P.cap_tokens));
  const int first = P.first_tokens ? max(0, P.first_tokens[s]) : 0;
  const int ptok = 16 * P.page_tiles;
  const int64_t col = (int64_t)(first / ptok) + nth;
  if (first >= ctx || col * ptok >= ctx) return;
  const int page = P.block_tables[(int64_t)table_row(P.seq_rows, s, P.bt_rows) * P.bt_stride + col];
  if (page < 0 || page >= P.n_pages) {
    if (lane == 0) flag_misuse(P.err, MISUSE_PAGE_OUT_OF_POOL);
    return;
  }
  const int nt = min(ptok, ctx - (int)col * ptok);
  const int tok = I8 ? (T == 128 ? lane >> 2 : (lane >> 1) & 15) : lane / LPT;  // of a load

  constexpr uint32_t kLeast = PK ? 0x80008000u : 0x80000000u, kMost = PK ? 0x7FFF7FFFu : 0x7FFFFFFFu;
  uint32_t lo[NW], hi[NW];
  float flo[NO], fhi[NO];
  bool ok = true;  // every key is finite
#pragma unroll
  for (int d = 0; d < NO; ++d) { flo[d] = kInf; fhi[d] = -kInf; }
  const auto clear = [&] {
#pragma unroll
    for (int i = 0; i < NW; ++i) { lo[i] = kMost; hi[i] = kLeast; }
  };
  // the tokens' lanes joined, and the lane's dims as floats
  const auto join = [&](float scale) {
    if constexpr (R32) fold_lanes<PK, NW, 32>(lo, hi);
    if constexpr (R16) fold_lanes<PK, N1, 16>(lo, hi);
    join_row<PK, LPT, NF>(lo, hi);
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const uint32_t w = side ? hi[i] : lo[i];
        float* f = side ? fhi : flo;
        const auto take = [&](int d, float x) { f[d] = side ? fmaxf(f[d], x) : fminf(f[d], x); };
        if constexpr (BLK) {  // words of the even, then of the odd dims of four
          take(4 * (i / 2) + i % 2, (float)((int)(w << 16) >> 24) * scale);
          take(4 * (i / 2) + i % 2 + 2, (float)((int)w >> 24) * scale);
        } else if constexpr (PK) {
          const uint32_t x = ordered_f16x2(w);
          f[2 * i] = half_lo(x);
          f[2 * i + 1] = half_hi(x);
        } else {
          f[i] = bitcast<float>(ordered_f32(w));
        }
      }
  };
  clear();
  for (int t = 0; t * BS < nt; ++t) {
    const int64_t tile = ((int64_t)page * P.page_tiles + t) * P.n_kv_heads + kvh;
    const uint8_t* base = P.kc + tile * P.tile_bytes;
    u32x4 c[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) c[j] = *reinterpret_cast<const u32x4*>(base + 1024 * j + 16 * lane);
    float scale = 1.0f;
    if constexpr (BLK) scale = half_lo(*reinterpret_cast<const uint32_t*>(P.ks + tile * kBlkScaleStep));
    if constexpr (REF) scale = reinterpret_cast<const float*>(P.ks + tile * P.stile_bytes)[tok];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int w0 = NS == 2 ? j * (NW / 2) : 0;
      const bool in = t * BS + (I8 ? tok : j * (WAVE / LPT) + tok) < nt;
#pragma unroll
      for (int i = 0; i < NW / NS; ++i) {
        uint32_t x;
        if constexpr (BLK) x = i % 2 ? c[j][i / 2] : bitcast<uint32_t>(bitcast<short2v>(c[j][i / 2]) << (short)8);  // codes in the high bytes
        else if constexpr (REF) x = ordered_f32(bitcast<uint32_t>(byte_to_f(c[j][i / 4], i % 4) * scale));
        else if constexpr (PK) x = ordered_f16x2(c[j][i]);
        else x = ordered_f32(c[j][i]);
        lo[w0 + i] = word_min<PK>(lo[w0 + i], in ? x : kMost);
        hi[w0 + i] = word_max<PK>(hi[w0 + i], in ? x : kLeast);
      }
    }
    if constexpr (BLK) {  // a scale a tile
      ok = ok && finite(scale);
      join(scale);
      clear();
    }
  }
  if constexpr (!BLK) join(1.0f);
  float top = 0.0f;
#pragma unroll
  for (int d = 0; d < NO; ++d) {
    top = fmaxf(top, fmaxf(fabsf(flo[d]), fabsf(fhi[d])));
    ok = ok && finite(flo[d]) && finite(fhi[d]);
  }
  top = wave_max(top);
  ok = __builtin_amdgcn_ballot_w64(!ok) == 0;
  const float inv = ok ? code_scale(top) : 0.0f;
  const int64_t at = (int64_t)page * P.n_kv_heads + kvh;
  // the first dim of the lane's: of its chunk, then the half that an exchange left it
  int dim = I8 ? (T == 128 ? 32 * (lane & 3) : 32 * (lane & 1) + 16 * (lane >> 5)) : EPC * (lane % LPT);
  if constexpr (R32) dim += (lane >> 5) * (N1 * (PK ? 2 : 1));
  if constexpr (R16) dim += ((lane >> 4) & 1) * NO;
  // of a row's lanes that hold the same dims the first writes the lower bounds and the
  // second the upper; where there is one (LPT >= 16) it writes both
  constexpr int WL = LPT < 16 ? LPT : 16;
  const int copy = (lane & 15) / WL;
  const auto write = [&](const float(&f)[NO], int8_t* dst) {
    uint32_t w[(NO + 3) / 4] = {};
#pragma unroll
    for (int d = 0; d < NO; ++d) w[d / 4] |= ((uint32_t)to_code(f[d], inv) & 0xFFu) << (8 * (d % 4));
    if constexpr (NO == 1) {
      *dst = (int8_t)w[0];
    } else if constexpr (NO == 2) {
      *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w[0];
    } else {
#pragma unroll
      for (int i = 0; i < NO / 4; ++i) reinterpret_cast<uint32_t*>(dst)[i] = w[i];
    }
  };
  int8_t* codes = P.codes + at * 2 * T + dim;
  if constexpr (WL == 16) {
    write(flo, codes);
    write(fhi, codes + T);
  } else if (copy < 2) {
    float f[NO];
#pragma unroll
    for (int d = 0; d < NO; ++d) f[d] = copy ? fhi[d] : flo[d];
    write(f, codes + copy * T);
  }
  if (lane == 0) P.scales[at] = ok ? top / 127.0f : kInf;
}

// The bounds of listed pages as fp32: four dims a thread.
DEV void index_read(const IndexReadParams& P) {
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= P.n_chunks) return;
  const uint32_t per = (uint32_t)P.io_hd / 4, row = i / per, at_page = row / (uint32_t)P.n_kv_heads;
  const int dim = (int)(i - row * per) * 4, kvh = (int)(row - at_page * (uint32_t)P.n_kv_heads);
  const int page = P.pages[at_page];
  float4 lo = make_float4(0, 0, 0, 0), hi = lo;
  if (page < 0 || page >= P.n_pages) {
    flag_misuse(P.err, MISUSE_PAGE_OUT_OF_POOL);
  } else {
    const int64_t at = (int64_t)page * P.n_kv_heads + kvh;
    const float scale = P.scales[at];
    const uint32_t* c = reinterpret_cast<const uint32_t*>(P.codes + at * 2 * P.tile_hd + dim);
    const uint32_t a = c[0], b = c[P.tile_hd / 4];
    if (scale < kInf) {
      lo = make_float4(byte_to_f(a, 0) * scale, byte_to_f(a, 1) * scale, byte_to_f(a, 2) * scale, byte_to_f(a, 3) * scale);
      hi = make_float4(byte_to_f(b, 0) * scale, byte_to_f(b, 1) * scale, byte_to_f(b, 2) * scale, byte_to_f(b, 3) * scale);
    } else {
      lo = make_float4(-kInf, -kInf, -kInf, -kInf);
      hi = make_float4(kInf, kInf, kInf, kInf);
    }
  }
  reinterpret_cast<float4*>(P.lower)[i] = lo;
  reinterpret_cast<float4*>(P.upper)[i] = hi;
}

// =============================================================================
// Selection. Over a page q . k is at most sum_d max(q_d lo_d, q_d hi_d) =
// [min(q, 0), max(q, 0)] . [lo, hi], a product over 2 T dims. Here q and the bounds are
// int8 codes, each the nearest: an estimate of that sum, not a bound. The codes' own sum
// is exact on v_mfma_i32_16x16x64_i8 (at most 128 x 127 x 127 < 2^24: exact in fp32 too),
// and the score
//     max over the group's heads of fp32(fp32(dot * page scale) * head scale)
// has the same bits however it is computed. Scores are kept as ordered 32-bit keys
// (larger key = chosen earlier). The pages that are always kept are not scored.
//
// Where a (sequence, KV head)'s scores fit LDS one workgroup computes them and selects
// (vk_page_select); longer contexts, and long ones of few sequences, are scored by
// several workgroups that leave the keys in memory (vk_page_scores) for a second launch
// (vk_page_topk).
//
// Bound: the rate at which rows of 2 T codes at unrelated addresses arrive. 64 sequences
// of 512 pages x 8 heads (T = 128), 69 MB: 15.8 us where the last-level cache holds the
// codes (as calls on one layer leave them), 19.3 from HBM, 3.6 TB/s; 32 of 2048, 136 MB: 27.7
// and 35. One sequence of 375 pages: 6.7 and 7.5 us, of which an empty launch is 4.7.
// =============================================================================

// What a workgroup of the selection knows of its (sequence, KV head).
struct SelUnit {
  int s, kvh, np, lo, n;   // pages of the context; the scored ones are [lo, lo + n)
  const int32_t* bt;
};
DEV SelUnit sel_unit(const SelectParams& P, int unit) {
  SelUnit u;
  u.kvh = unit % P.n_kv_heads;
  u.s = unit / P.n_kv_heads;
  const int ctx = max(0, min(P.context_lens[u.s], P.cap_tokens));
  u.np = (int)(((uint32_t)ctx + (uint32_t)P.page_tokens - 1) / (uint32_t)P.page_tokens);  // ctx ends at 2^31 - 1
  u.lo = P.n_first;
  u.n = u.np > P.n_list ? u.np - P.n_first - P.n_last : 0;  // none: all pages are listed
  u.bt = P.block_tables + (int64_t)table_row(P.seq_rows, u.s, P.bt_rows) * P.bt_stride;
  return u;
}

// Values of query row r of a (sequence, KV head): dims EPL l .. of lane l, rows past the
// group as its last one.
template <int QT, int T>
DEV void load_query_row(const SelectParams& P, int unit, int r, float (&x)[T / WAVE]) {
  constexpr int EPL = T / WAVE;
  const int G = P.n_heads / P.n_kv_heads;
  const int64_t row = ((int64_t)unit * G + min(r, G - 1)) * P.io_hd;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    const int64_t at = row + min(lane_id() * EPL + e, P.io_hd - 1);
    x[e] = QT == DT_F32 ? reinterpret_cast<const float*>(P.q)[at] : h2f(reinterpret_cast<const uint16_t*>(P.q)[at]);
  }
}
// Codes of the (sequence, KV head)'s queries in LDS, negative parts first. x: row w of wave w,
// which is loaded ahead of everything else. Ends with a barrier.
template <int QT, int T>
DEV void query_codes(const SelectParams& P, int unit, float (&x)[T / WAVE], int8_t (*qc)[2 * T], float* qs) {
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE, G = P.n_heads / P.n_kv_heads;
  constexpr int EPL = T / WAVE;
  for (int r = w; r < G; r += kSelWaves) {
    if (r != w) load_query_row<QT, T>(P, unit, r, x);
    float bad = 0.0f, top = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      x[e] = lane * EPL + e < P.io_hd ? x[e] : 0.0f;
      top = fmaxf(top, fabsf(x[e]));
      bad = fmaf(x[e], 0.0f, bad);
    }
    top = wave_max(top);
    const bool ok = __builtin_amdgcn_ballot_w64(!(bad == 0.0f)) == 0;
    const float inv = ok ? code_scale(top) : 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int c = ok ? to_code(x[e], inv) : 0;
      qc[r][lane * EPL + e] = (int8_t)min(c, 0);
      qc[r][T + lane * EPL + e] = (int8_t)max(c, 0);
    }
    if (lane == 0) qs[r] = ok ? top / 127.0f : 0.0f;
  }
  __syncthreads();
}

// A wave's turn of 64 scored pages: their ids, codes and scales. keys[i] is page u.lo + i.
// Codes are loaded in the operands' order, or BY_ROW, a row by adjacent lanes (LPR each),
// and change lanes in LDS. A CU takes 36 GB/s in the operands' order, where adjacent lanes
// read 16 rows, and 95 by rows, so fewer (sequence, KV head)s than CUs load by rows (one
// sequence of 375 pages x 8 heads: 6.7 us against 7.3 in the operands' order, 8 of 512: 7.2
// against 8.5, 31 of 512: 8.9 either way); the operands' order takes fewer registers and no
// LDS, so that more workgroups share a CU (64 sequences of 512 pages: 15.8 us against 20.3 by
// rows; 32 of 2048, a workgroup a CU, 27.7 against 26.5). The keys of long contexts of few
// (vk_page_scores) are loaded in the operands' order too; by rows is not built there.
template <int T, bool BY_ROW>
struct PageTurn {
  static constexpr int KJ = 2 * T / 64;                                         // products of 64 dims
  static constexpr int LPR = 2 * T / 16, RPL = WAVE / LPR, NL = WAVE / RPL;  // lanes a row, rows a load, loads
  int raw;              // the lane's page id
  u32x4 codes[NL];      // by rows: chunk lane % LPR of page i RPL + lane / LPR; else chunk 4 (i % KJ) + g of page 16 (i / KJ) + n
  float scale;
};
// LDS of one wave: 16 rows of 2 T codes, a row's 16-byte chunks in an order of its own so
// that reads of one chunk of all rows meet all banks.
template <int T>
struct RowTile {
  u32x4 c[16][2 * T / 16];
  static __device__ __forceinline__ int place(int row, int chunk) { return chunk ^ (row & (2 * T / 16 - 1)); }
};
DEV int page_id(const SelectParams& P, const SelUnit& u, int p) { return u.bt[u.lo + min(p + lane_id(), u.n - 1)]; }
template <int T, bool BY_ROW>
DEV void load_turn(const SelectParams& P, const SelUnit& u, int raw, PageTurn<T, BY_ROW>& t) {
  using Turn = PageTurn<T, BY_ROW>;
  const int lane = lane_id(), n = lane & 15, g = lane >> 4, page = min(max(raw, 0), P.n_pool_pages - 1);
  t.raw = raw;
  if constexpr (BY_ROW) {
#pragma unroll
    for (int i = 0; i < Turn::NL; ++i) {
      const int64_t at = (int64_t)__shfl(page, i * Turn::RPL + lane / Turn::LPR, WAVE) * P.n_kv_heads + u.kvh;
      t.codes[i] = *reinterpret_cast<const u32x4*>(P.codes + at * 2 * T + 16 * (lane % Turn::LPR));
    }
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t at = (int64_t)__shfl(page, 16 * v + n, WAVE) * P.n_kv_heads + u.kvh;
      const u32x4* c = reinterpret_cast<const u32x4*>(P.codes + at * 2 * T + 16 * g);
#pragma unroll
      for (int j = 0; j < Turn::KJ; ++j) t.codes[v * Turn::KJ + j] = c[4 * j];
    }
  }
  t.scale = P.scales[(int64_t)page * P.n_kv_heads + u.kvh];
}
// Pages 16 v .. 16 v + 15 of a turn as operands: chunk 4 j + g of page n.
template <int T, bool BY_ROW>
DEV void turn_operands(const PageTurn<T, BY_ROW>& t, int v, RowTile<T>* tile, i32x4 (&kb)[2 * T / 64]) {
  using Turn = PageTurn<T, BY_ROW>;
  const int lane = lane_id(), n = lane & 15, g = lane >> 4, r = lane / Turn::LPR, c = lane % Turn::LPR;
  if constexpr (BY_ROW) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < Turn::NL / 4; ++i) tile->c[i * Turn::RPL + r][RowTile<T>::place(i * Turn::RPL + r, c)] = t.codes[v * (Turn::NL / 4) + i];
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int j = 0; j < Turn::KJ; ++j) kb[j] = bitcast<i32x4>(BY_ROW ? tile->c[n][RowTile<T>::place(n, 4 * j + g)] : t.codes[v * Turn::KJ + j]);
}

// Keys of scored pages first, first + step, ..: 64 a turn, as four products of 16 pages
// (the pages are the columns, the heads the rows; rows past the group repeat its last one,
// whose scores change no maximum). The first turn's loads are issued before the queries'
// codes are made. Returns the lane's least and largest key.
template <int QT, int T, int RT, bool BY_ROW>
DEV uint2 score_pages(const SelectParams& P, const SelUnit& u, int unit, float (&x)[T / WAVE], int8_t (*qc)[2 * T], float* qs,
                      RowTile<T>* tile, int first, int step, uint32_t* keys) {
  constexpr int KJ = 2 * T / 64;  // products of 64 dims
  const int lane = lane_id(), n = lane & 15, g = lane >> 4;
  uint2 span = make_uint2(0xFFFFFFFFu, 0u);
  PageTurn<T, BY_ROW> t;
  int next = 0;
  if (first < u.n) {
    const int raw = page_id(P, u, first);
    next = page_id(P, u, first + step);
    load_turn<T, BY_ROW>(P, u, raw, t);
  }
  query_codes<QT, T>(P, unit, x, qc, qs);
  const int G = P.n_heads / P.n_kv_heads;
  if (first >= u.n) return span;
  i32x4 qa[RT][KJ];
  float qsc[RT][4];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int j = 0; j < KJ; ++j) qa[rt][j] = *reinterpret_cast<const i32x4*>(&qc[min(16 * rt + n, G - 1)][64 * j + 16 * g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) qsc[rt][i] = qs[min(16 * rt + 4 * g + i, G - 1)];
  }
  bool out = false;
  for (int p0 = first; p0 < u.n; p0 += step) {
    out |= t.raw < 0 || t.raw >= P.n_pool_pages;
    float best[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float sc = __shfl(t.scale, 16 * v + n, WAVE);
      i32x4 kb[KJ];
      turn_operands<T, BY_ROW>(t, v, tile, kb);
      best[v] = -kInf;  // a score that is not a number counts as this
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        i32x4 dot = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < KJ; ++j) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[rt][j], kb[j], dot, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) best[v] = fmaxf(best[v], ((float)dot[i] * sc) * qsc[rt][i]);
      }
    }
    const bool top = t.scale == kInf;
    if (p0 + step < u.n) {
      const int raw = next;
      next = page_id(P, u, p0 + 2 * step);
      load_turn<T, BY_ROW>(P, u, raw, t);
    }
    // the maximum over the row groups, which leaves lane l page p0 + l's
    swap_lanes<32>(best[0], best[2]);
    swap_lanes<32>(best[1], best[3]);
    float a = fmaxf(best[0], best[2]), b = fmaxf(best[1], best[3]);
    swap_lanes<16>(a, b);
    const uint32_t key = order_key(top ? kInf : fmaxf(a, b));
    if (p0 + lane < u.n) {
      keys[p0 + lane] = key;
      span.x = min(span.x, key);
      span.y = max(span.y, key);
    }
  }
  if (__builtin_amdgcn_ballot_w64(out) != 0 && lane == 0) flag_misuse(P.err, MISUSE_PAGE_OUT_OF_POOL);
  return span;
}

// Writes a (sequence, KV head)'s list: the kept pages and, of the scored ones, the
// `want` with the largest keys, ties to the lower page, in ascending order. The want-th
// largest key is found in rounds: the keys in question lie in [base, base + 2^bits);
// their 8 leading bits are counted, and the bin that holds the key sought is the next
// round's range. A bin of at most 64 keys is ranked by one wave.
struct SelScratch {
  int hist[256];
  int turn[kSelMaxWaves][2];
  uint32_t least, most, bin_keys[64];
  int n_bin, found[3];
};
DEV void select_begin(SelScratch& x) {  // before a barrier
  if (threadIdx.x == 0) { x.least = 0xFFFFFFFFu; x.most = 0; }
}
template <int W, typename Keys>
DEV void select_top(const SelectParams& P, const SelUnit& u, const Keys keys, uint2 span, int32_t* pages, SelScratch& x) {
  const int tid = (int)threadIdx.x, lane = lane_id(), w = tid / WAVE;
  const int want_all = P.n_list - P.n_first - P.n_last;
  for (int i = tid; i < P.n_first; i += W * WAVE) pages[i] = i;
  for (int i = tid; i < P.n_last; i += W * WAVE) pages[P.n_list - P.n_last + i] = u.np - P.n_last + i;
  if (want_all == 0) return;
  const uint32_t least = ~wave_max_u(~span.x), most = wave_max_u(span.y);
  if (lane == 0) { atomicMin(&x.least, least); atomicMax(&x.most, most); }
  __syncthreads();
  uint32_t base = x.least;
  const uint32_t range = x.most - base;
  int bits = range ? 32 - __builtin_clz(range) : 0, want = want_all;
  uint32_t key = base;  // the want_all-th largest, `want` of whose equals are listed
  while (bits > 0) {
    const int shift = max(0, bits - 8);
    if (tid < 256) x.hist[tid] = 0;
    if (tid == 0) x.n_bin = 0;
    __syncthreads();
    for (int i = tid; i < u.n; i += W * WAVE) {
      const uint32_t k = keys[i] - base;
      if (bits == 32 || k >> bits == 0) atomicAdd(&x.hist[k >> shift], 1);
    }
    __syncthreads();
    if (w == 0) {  // bins 255 - 4 l - e of lane l, largest first
      int c[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) { c[e] = x.hist[255 - 4 * lane - e]; sum += c[e]; }
      const int incl = wave_prefix_sum(sum);
      int before = incl - sum;
      if (before < want && incl >= want) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (before < want && before + c[e] >= want) {
            x.found[0] = 255 - 4 * lane - e;
            x.found[1] = want - before;
            x.found[2] = c[e];
            before = want;  // no later bin
          } else {
            before += c[e];
          }
        }
      }
    }
    __syncthreads();
    base += (uint32_t)x.found[0] << shift;
    want = x.found[1];
    key = base;
    bits = shift;
    const int m = x.found[2];
    if (bits == 0) break;  // the bin is one key
    if (m > WAVE) { __syncthreads(); continue; }
    // the m keys of the bin
    for (int i = tid; i < u.n; i += W * WAVE) {
      const uint32_t k = keys[i];
      if ((k - base) >> bits == 0) x.bin_keys[atomicAdd(&x.n_bin, 1)] = k;
    }
    __syncthreads();
    // the largest that `want` of them reach
    const uint32_t mine = lane < m ? x.bin_keys[lane] : 0;
    int reach = 0;
    for (int j = 0; j < m; j += 8)  // (lanes past the m hold 0, which no key is)
#pragma unroll
      for (int e = 0; e < 8; ++e) reach += (uint32_t)readlane_i((int)mine, j + e) >= mine;
    key = wave_max_u(lane < m && reach >= want ? mine : 0);
    want -= __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine > key));
    break;
  }
  __syncthreads();
  // a wave's share of the pages is one run of them, so that its place in the list follows
  // from how many the waves before it list
  const int per = (u.n + W * WAVE - 1) / (W * WAVE) * WAVE;
  const int i0 = w * per, i1 = min(u.n, i0 + per);
  int above = 0, equal = 0;
  for (int i = i0 + lane; i - lane < i1; i += WAVE) {
    const uint32_t k = i < i1 ? keys[i] : 0;
    above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < i1 && k > key));
    equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < i1 && k == key));
  }
  if (lane == 0) { x.turn[w][0] = above; x.turn[w][1] = equal; }
  __syncthreads();
  above = equal = 0;
  for (int v = 0; v < w; ++v) { above += x.turn[v][0]; equal += x.turn[v][1]; }
  pages += P.n_first;
  for (int i = i0 + lane; i - lane < i1; i += WAVE) {
    const uint32_t k = i < i1 ? keys[i] : 0;
    const uint64_t gt = __builtin_amdgcn_ballot_w64(i < i1 && k > key), eq = __builtin_amdgcn_ballot_w64(i < i1 && k == key);
    const uint64_t below = (1ull << lane) - 1;
    const int e = equal + __builtin_popcountll(eq & below);
    if (i < i1 && (k > key || (k == key && e < want))) pages[above + __builtin_popcountll(gt & below) + min(e, want)] = u.lo + i;
    above += __builtin_popcountll(gt);
    equal += __builtin_popcountll(eq);
  }
}

// A context of no more pages than the list has places: all of them.
template <int W>
DEV void list_all(const SelectParams& P, const SelUnit& u, int32_t* pages) {
  for (int i = (int)threadIdx.x; i < P.n_list; i += W * WAVE) pages[i] = i < u.np ? i : -1;
}

// The wave's first page of a workgroup's chunk.
constexpr int kSelThreads = kSelWaves * WAVE;
DEV int first_page(int chunk) { return chunk * kSelThreads + __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE) * WAVE; }

template <int QT, int T, int RT, bool BY_ROW>
DEV void page_select(const SelectParams& P) {
  __shared__ __align__(16) int8_t qc[16 * RT][2 * T];
  __shared__ float qs[16 * RT];
  __shared__ RowTile<T> tiles[BY_ROW ? kSelWaves : 1];
  __shared__ uint32_t keys[kSelPages];
  __shared__ SelScratch scratch;
  // each XCD takes a run of the units, so that the heads of a sequence, whose rows lie side by
  // side, are read through one cache (64 sequences of 512 pages: 0.9 us less)
  const int units = P.n_seqs * P.n_kv_heads, run = units / 8, b = (int)blockIdx.x;
  const int unit = b < 8 * run ? (b & 7) * run + (b >> 3) : b;
  float x[T / WAVE];
  load_query_row<QT, T>(P, unit, (int)threadIdx.x / WAVE, x);
  const SelUnit u = sel_unit(P, unit);
  int32_t* pages = P.pages + (int64_t)unit * P.n_list;
  if (u.n == 0) {
    list_all<kSelWaves>(P, u, pages);
    return;
  }
  select_begin(scratch);
  const uint2 span = score_pages<QT, T, RT, BY_ROW>(P, u, unit, x, qc, qs, &tiles[BY_ROW ? threadIdx.x / WAVE : 0], first_page(0), kSelThreads, keys);
  select_top<kSelWaves>(P, u, keys, span, pages, scratch);
}

template <int QT, int T, int RT>
DEV void page_scores(const SelectParams& P) {
  __shared__ __align__(16) int8_t qc[16 * RT][2 * T];
  __shared__ float qs[16 * RT];
  const int chunk = (int)(blockIdx.x % P.n_chunks), unit = (int)(blockIdx.x / P.n_chunks);
  float x[T / WAVE];
  load_query_row<QT, T>(P, unit, (int)threadIdx.x / WAVE, x);
  const SelUnit u = sel_unit(P, unit);
  if (chunk * kSelThreads >= u.n) return;
  score_pages<QT, T, RT, false>(P, u, unit, x, qc, qs, nullptr, first_page(chunk), P.n_chunks * kSelThreads, P.keys + (int64_t)unit * P.max_pages);
}
template <int W>
DEV void page_topk(const SelectParams& P) {
  __shared__ SelScratch scratch;
  const SelUnit u = sel_unit(P, (int)blockIdx.x);
  int32_t* pages = P.pages + (int64_t)blockIdx.x * P.n_list;
  if (u.n == 0) {
    list_all<W>(P, u, pages);
    return;
  }
  const uint32_t* keys = P.keys + (int64_t)blockIdx.x * P.max_pages;
  select_begin(scratch);
  uint2 span = make_uint2(0xFFFFFFFFu, 0u);
  for (int i = (int)threadIdx.x; i < u.n; i += W * WAVE) {
    const uint32_t k = keys[i];
    span = make_uint2(min(span.x, k), max(span.y, k));
  }
  __syncthreads();
  select_top<W>(P, u, keys, span, pages, scratch);
}

// =============================================================================
// Attention of one query row per head over listed pages:
//     out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t),
// over the tokens below the context's end of the pages that the list names. One
// workgroup per (sequence, KV head, part of its list): it stages the part's pages
// in LDS, its waves take pairs of 16-token tiles in turn, each with a running
// maximum of its own, and the waves' sums meet in LDS. Scores are S^T = K q^T and
// values O^T = V^T p^T on the matrix cores: the lane that gets the scores of query
// row n and tokens 4 g .. 4 g + 3 holds exactly the operand of the value product.
// p enters it as two fp16 parts, p = hi + lo to 2^-22 relative (fp32 pools: fp32
// throughout); the maximum is that of p times the value's scale, so that what is
// rounded to fp16 lies in (0, 2^15].
// Bound: HBM where the (sequence, KV head)s fill the CUs. 64 sequences of 64 listed pages x
// 8 heads, a call from HBM: fp16 47.8 us, 270 MB at 5.7 TB/s; fp32 92.4 us, 5.8 TB/s; int8 of
// a scale per token 29.8 us, 4.7 TB/s, and per tile 29.2 us, 4.7 TB/s, with the launch and the
// chain of list, table and first tile. Few sequences: that chain, then the merge (one
// sequence of 64 pages: 7.1 + 3.3 us).
// =============================================================================
constexpr float kShift = 11.0f;           // p is held times 2^11: fp16 subnormals begin 2^-36 below the largest
constexpr float kRaise = 4.0f;            // the maximum is raised when a score passes it by 2^4
constexpr float kMinScale = 0x1p-80f;     // value scales below this do not lower the maximum further
constexpr int kSparseMaxWaves = 8;

template <int KV, int T>
struct SparseTile {
  static constexpr int W = 16 * T * Esz<KV>::v / 256;  // registers of a K or V tile
  DW<W> k, v;
  float ks[4], vs[4];  // I8_REF: scales of tokens 4 g .. 4 g + 3; I8_BLK: the tile's in [0]
  int n_tok;           // tokens below the context's end
};

// Issues the loads of tile t of the unit's list (none past the last: zeros, no traffic).
template <int KV, int T>
DEV void sparse_load(SparseTile<KV, T>& st, const SparseParams& P, const int* page, const int* pos, int n_tiles, int t, int ctx, int kvh) {
  constexpr int ESZ = Esz<KV>::v;
  const int lane = lane_id(), n = lane & 15, g = lane >> 4;
  const int e = min(t, n_tiles - 1) / P.page_tiles, sub = min(t, n_tiles - 1) - e * P.page_tiles;
  const int start = __builtin_amdgcn_readfirstlane(pos[e]) + 16 * sub;
  st.n_tok = t < n_tiles ? min(16, ctx - start) : 0;
  const int64_t tile = ((int64_t)__builtin_amdgcn_readfirstlane(page[e]) * P.page_tiles + sub) * P.n_kv_heads + kvh;
  const uint32_t bytes = st.n_tok > 0 ? P.tile_bytes : 0u;
  const rsrc_t kr = make_rsrc(P.kc + tile * P.tile_bytes, bytes), vr = make_rsrc(P.vc + tile * P.tile_bytes, bytes);
  constexpr int KP = T * ESZ / 64;  // 16-byte pieces of a lane's K
#pragma unroll
  for (int j = 0; j < KP; ++j) {
    uint32_t off;
    if constexpr (ESZ == 1)  // [2][16][T / 32][16]: T = 128: half j, slice g; T = 64: half g / 2, slice g % 2
      off = T == 128 ? 1024 * j + 64 * n + 16 * g : 512 * (g >> 1) + 32 * n + 16 * (g & 1);
    else if constexpr (ESZ == 2)
      off = 2 * T * n + 64 * j + 16 * g;
    else
      off = 4 * T * n + 64 * j + 16 * g;
    const DW<4> x = buf_load<4>(kr, off);
#pragma unroll
    for (int i = 0; i < 4; ++i) st.k.d[4 * j + i] = x.d[i];
  }
  // V [8][T][2]: token pairs 2 g and 2 g + 1
  if constexpr (ESZ == 1 && T == 64) {
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      const DW<2> x = buf_load<2>(vr, (2 * g + pr) * 2 * T + 8 * n);
      st.v.d[2 * pr] = x.d[0];
      st.v.d[2 * pr + 1] = x.d[1];
    }
  } else {
    constexpr int VP = T * ESZ * 2 / 256;  // pieces of a token pair's row
#pragma unroll
    for (int h = 0; h < VP; ++h)
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        const DW<4> x = buf_load<4>(vr, (2 * g + pr) * 2 * T * ESZ + 256 * h + 16 * n);
#pragma unroll
        for (int i = 0; i < 4; ++i) st.v.d[8 * h + 4 * pr + i] = x.d[i];
      }
  }
  if constexpr (KV == KV_I8_REF) {
    const uint32_t sb = st.n_tok > 0 ? P.stile_bytes : 0u;
    const DW<4> a = buf_load<4, 0>(make_rsrc(P.ks + tile * P.stile_bytes, sb), 16 * g);
    const DW<4> b = buf_load<4, 0>(make_rsrc(P.vs + tile * P.stile_bytes, sb), 16 * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) { st.ks[i] = bitcast<float>(a.d[i]); st.vs[i] = bitcast<float>(b.d[i]); }
  }
  if constexpr (KV == KV_I8_BLK) {
    const DW<1> a = buf_load<1, 0>(make_rsrc(P.ks + tile * kBlkScaleStep, st.n_tok > 0 ? 4u : 0u), 0);
    st.ks[0] = half_lo(a.d[0]);
    st.vs[0] = half_hi(a.d[0]);
  }
}

// 8 fp16 values of the K operand's chunk j.
template <int KV, int T>
DEV half8 sparse_k(const SparseTile<KV, T>& st, int j) {
  uint4 x;
  if constexpr (Esz<KV>::v == 1) {
    i8x4_to_h2x2(st.k.d[2 * j], x.x, x.y);
    i8x4_to_h2x2(st.k.d[2 * j + 1], x.z, x.w);
  } else {
    x = make_uint4(st.k.d[4 * j], st.k.d[4 * j + 1], st.k.d[4 * j + 2], st.k.d[4 * j + 3]);
  }
  return bitcast<half8>(x);
}
// Token pair words (fp16 even, odd) of dim tile i: pair 2 g, pair 2 g + 1. Values of
// tokens past the context's end are zero whatever the pool holds there (it may be
// infinite or NaN; they meet p = 0).
template <int KV, int T>
DEV uint2 sparse_v(const SparseTile<KV, T>& st, int i) {
  if constexpr (Esz<KV>::v == 1) {
    constexpr int WPP = T / 32;  // words of a pair's row that a lane holds, two dims each
    uint2 a, b;
    i8x4_to_h2x2(st.v.d[i / 2], a.x, a.y);
    i8x4_to_h2x2(st.v.d[WPP + i / 2], b.x, b.y);
    return i % 2 ? make_uint2(a.y, b.y) : make_uint2(a.x, b.x);
  } else {
    const int left = st.n_tok - 4 * (lane_id() >> 4);  // of the lane's four tokens
    const uint32_t a = (left > 0 ? 0xFFFFu : 0u) | (left > 1 ? 0xFFFF0000u : 0u);
    const uint32_t b = (left > 2 ? 0xFFFFu : 0u) | (left > 3 ? 0xFFFF0000u : 0u);
    return make_uint2(st.v.d[8 * (i / 4) + i % 4] & a, st.v.d[8 * (i / 4) + 4 + i % 4] & b);
  }
}
// Dim that row 4 g + r of dim tile i holds.
template <int KV, int T>
DEV int sparse_dim(int i, int g, int r) {
  if constexpr (Esz<KV>::v == 1) return T == 128 ? 8 * (4 * g + r) + i : 4 * (4 * g + r) + i;
  else if constexpr (Esz<KV>::v == 2) return 64 * (i / 4) + 4 * (4 * g + r) + i % 4;
  else return 32 * (i / 2) + 2 * (4 * g + r) + i % 2;
}
// First dim of the query's chunk j (8 dims) of lane group g, as sparse_k has K's.
template <int KV, int T>
DEV int sparse_qdim(int j, int g) {
  if constexpr (Esz<KV>::v == 1) return T == 128 ? 32 * g + 8 * j : 32 * (g & 1) + 16 * (g >> 1) + 8 * j;
  else return 32 * j + 8 * g;
}

// N query values, wherever they start, as they are stored.
template <int QT, int N>
struct QueryWords {
  typedef uint32_t words __attribute__((ext_vector_type(QT == DT_F32 ? N : N / 2), aligned(2)));
  words r;
  __device__ __forceinline__ void load(const void* q, int64_t at) { r = *reinterpret_cast<const words*>(reinterpret_cast<const uint8_t*>(q) + at * (QT == DT_F32 ? 4 : 2)); }
  __device__ __forceinline__ float value(int i) const { return QT == DT_F32 ? bitcast<float>(r[i]) : i % 2 ? half_hi(r[i / 2]) : half_lo(r[i / 2]); }
};

template <int KV, int QT, int T, int RT>
DEV void sparse_attn(const SparseParams& P) {
  constexpr bool F32 = KV == KV_F32, BLK = KV == KV_I8_BLK, REF = KV == KV_I8_REF;
  constexpr int CH = F32 ? 1 : 2;   // tiles taken at once
  constexpr int KC = T / 32;        // score products of a tile (fp16 operands)
  constexpr int NT = T / 16;        // dim tiles
  constexpr bool QSPLIT = !F32 && QT == DT_F32;
  constexpr int MW = RT == 1 ? kSparseMaxWaves : kSparseMaxWaves / 2;
  __shared__ int page[kSparseEntries], pos[kSparseEntries];
  __shared__ float wacc[MW][16 * RT][T];
  __shared__ float wml[MW][16 * RT][2];
  __shared__ int n_valid;
  const int tid = (int)threadIdx.x, lane = lane_id(), n = lane & 15, g = lane >> 4, nw = (int)blockDim.x / WAVE;
  const int w = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int split = (int)(blockIdx.x % P.n_splits), unit = (int)(blockIdx.x / P.n_splits);
  const int kvh = unit % P.n_kv_heads, s = unit / P.n_kv_heads;
  const int G = P.n_heads / P.n_kv_heads;
  const int ctx = max(0, min(P.context_lens[s], P.cap_tokens));
  const int64_t row0 = (int64_t)s * P.n_heads + (int64_t)kvh * G;

  // the list's loads, then the queries', are under way before anything waits: the list's lead
  // to the tiles
  const int32_t* list = P.pages + (int64_t)unit * P.n_list;
  const int first = split * P.split_entries, e1 = min(P.n_list, first + P.split_entries);
  const int ahead = list[min(first + lane, e1 - 1)];
  // q^T: row n of each 16-row tile (rows past the group repeat its last one: their columns of
  // the results are not used), zeros past head_dim
  constexpr int QN = F32 ? 4 : 8, QC = F32 ? T / 16 : KC;  // values of a chunk, chunks
  const auto qdim = [&](int j) { return F32 ? 16 * j + 4 * g : sparse_qdim<KV, T>(j, g); };
  QueryWords<QT, QN> qw[RT][QC];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int j = 0; j < QC; ++j)
      qw[rt][j].load(P.q, (row0 + min(16 * rt + n, G - 1)) * P.io_hd + min(qdim(j), P.io_hd - QN));

  if (w == 0) {  // the part's entries that name a page of the context
    const int32_t* bt = P.block_tables + (int64_t)table_row(P.seq_rows, s, P.bt_rows) * P.bt_stride;
    const int ptok = 16 * P.page_tiles;
    int count = 0;
    bool bad = false;
    for (int e0 = first; e0 < e1; e0 += WAVE) {
      const int col = e0 + lane < e1 ? (e0 == first ? ahead : list[e0 + lane]) : -1;
      const bool in = col >= 0 && (int64_t)col * ptok < ctx;
      const int raw = in ? bt[col] : 0;
      bad |= raw < 0 || raw >= P.n_pages;
      const uint64_t m = __builtin_amdgcn_ballot_w64(in);
      if (in) {
        const int at = count + __builtin_popcountll(m & ((1ull << lane) - 1));
        page[at] = min(max(raw, 0), P.n_pages - 1);
        pos[at] = col * ptok;
      }
      count += __builtin_popcountll(m);
    }
    if (lane == 0) n_valid = count;
    if (__builtin_amdgcn_ballot_w64(bad) != 0 && lane == 0) flag_misuse(P.err, MISUSE_PAGE_OUT_OF_POOL);
  }

  half8 qa[RT][F32 ? 1 : KC], qlo[RT][QSPLIT ? KC : 1];
  float qf[RT][F32 ? T / 4 : 1], scale_log2[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    scale_log2[rt] = P.scale_log2;
    float top = 0.0f;
    if constexpr (QSPLIT) {
#pragma unroll
      for (int j = 0; j < QC; ++j)
#pragma unroll
        for (int i = 0; i < QN; ++i) top = fmaxf(top, qdim(j) < P.io_hd ? fabsf(qw[rt][j].value(i)) : 0.0f);
    }
    int up = 0;  // an fp32 row is taken times 2^up, which brings its largest to [2^13, 2^14): fp16 ends at 2^16
    if constexpr (QSPLIT) {
      top = fmaxf(top, shfl_xor(top, 16));
      top = fmaxf(top, shfl_xor(top, 32));
      up = top > 0.0f && top < kInf ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
      scale_log2[rt] = __builtin_amdgcn_ldexpf(P.scale_log2, -up);
    }
#pragma unroll
    for (int j = 0; j < QC; ++j)
#pragma unroll
      for (int i = 0; i < QN; ++i) {
        const float x = qdim(j) < P.io_hd ? qw[rt][j].value(i) : 0.0f;
        if constexpr (F32) {
          qf[rt][QN * j + i] = x;
        } else {
          const float v = QSPLIT ? __builtin_amdgcn_ldexpf(x, up) : x;
          qa[rt][j][i] = (_Float16)v;
          if constexpr (QSPLIT) qlo[rt][j][i] = (_Float16)(v - (float)qa[rt][j][i]);
        }
      }
  }
  __syncthreads();
  const int n_tiles = __builtin_amdgcn_readfirstlane(n_valid) * P.page_tiles;

  f32x4 acc[RT][NT];
  float M[RT], L[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    M[rt] = -kInf;
    L[rt] = 0.0f;
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[rt][i] = f32x4{0, 0, 0, 0};
  }

  auto step = [&](SparseTile<KV, T>(&st)[CH]) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[CH][4];
      float top = -kInf;
#pragma unroll
      for (int u = 0; u < CH; ++u) {
        f32x4 sc = {0, 0, 0, 0};
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < T / 4; ++j) sc = __builtin_amdgcn_mfma_f32_16x16x4f32(bitcast<float>(st[u].k.d[j]), qf[rt][j], sc, 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < KC; ++j) {
            const half8 k = sparse_k<KV, T>(st[u], j);
            sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qa[rt][j], sc, 0, 0, 0);
            if constexpr (QSPLIT) sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qlo[rt][j], sc, 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = sc[i] * scale_log2[rt], up = 0.0f;
          if constexpr (BLK) { v = sc[i] * st[u].ks[0] * scale_log2[rt]; up = __builtin_amdgcn_logf(fmaxf(st[u].vs[0], kMinScale)); }
          if constexpr (REF) { v = sc[i] * st[u].ks[i] * scale_log2[rt]; up = __builtin_amdgcn_logf(fmaxf(st[u].vs[i], kMinScale)); }
          x[u][i] = 4 * g + i < st[u].n_tok ? v : -kInf;
          top = fmaxf(top, x[u][i] + up);
        }
      }
      top = fmaxf(top, shfl_xor(top, 16));
      top = fmaxf(top, shfl_xor(top, 32));
      const bool raise = top > M[rt] + kRaise;
      if (__builtin_amdgcn_ballot_w64(raise) != 0) {
        const float m = raise ? top : M[rt];
        const float f = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(M[rt] - m);
        M[rt] = m;
        L[rt] *= f;
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[rt][i] *= f;
      }
      float p[CH][4];
      half8 hi, lo;
#pragma unroll
      for (int u = 0; u < CH; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[u][i] = x[u][i] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(x[u][i] - M[rt] + (F32 ? 0.0f : kShift));
          L[rt] += p[u][i];
          if constexpr (BLK) p[u][i] *= st[u].n_tok > 0 ? st[u].vs[0] : 0.0f;
          if constexpr (REF) p[u][i] *= 4 * g + i < st[u].n_tok ? st[u].vs[i] : 0.0f;
          if constexpr (!F32) {
            // hi is cut, not rounded: the compiler fuses the scale's product into one of two
            // roundings, and where the two differ lo is not the rest (2^-11 of the token's weight)
            const float cut = bitcast<float>(bitcast<uint32_t>(p[u][i]) & 0xFFFFE000u);
            hi[4 * u + i] = (_Float16)cut;
            lo[4 * u + i] = (_Float16)(p[u][i] - cut);
          }
        }
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) {  // token 4 g + t: word (dim i % 2, token t % 2) of pair 2 g + t / 2
            const uint32_t v = 4 * g + t < st[0].n_tok ? st[0].v.d[8 * (i / 2) + 4 * (t / 2) + 2 * (i % 2) + t % 2] : 0u;
            acc[rt][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(bitcast<float>(v), p[0][t], acc[rt][i], 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint2 a = sparse_v<KV, T>(st[0], i), b = sparse_v<KV, T>(st[CH - 1], i);
          const half8 v = bitcast<half8>(make_uint4(a.x, a.y, b.x, b.y));
          acc[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi, acc[rt][i], 0, 0, 0);
          acc[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo, acc[rt][i], 0, 0, 0);
        }
      }
    }
  };

  if (n_tiles > 0) {
    SparseTile<KV, T> a[CH], b[CH];
    const auto load = [&](SparseTile<KV, T>(&st)[CH], int c) {
#pragma unroll
      for (int u = 0; u < CH; ++u) sparse_load<KV, T>(st[u], P, page, pos, n_tiles, c * CH + u, ctx, kvh);
    };
    const int n_chunks = (n_tiles + CH - 1) / CH;
    int c = w;
    load(a, c);
    for (; c < n_chunks; c += 2 * nw) {
      load(b, c + nw);
      step(a);
      if (c + nw >= n_chunks) break;
      load(a, c + 2 * nw);
      step(b);
    }
  }

  // the waves' sums: out = sum_w 2^(M_w - M) acc_w / sum_w 2^(M_w - M) L_w
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    L[rt] += shfl_xor(L[rt], 16);
    L[rt] += shfl_xor(L[rt], 32);
    const int r = 16 * rt + n;
    if (r < G) {
      if (g == 0) { wml[w][r][0] = M[rt]; wml[w][r][1] = L[rt]; }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) wacc[w][r][sparse_dim<KV, T>(i, g, k)] = acc[rt][i][k];
    }
  }
  __syncthreads();
  for (int e = tid; e < G * T; e += (int)blockDim.x) {
    const int r = e / T, d = e % T;
    float m = -kInf, l = 0.0f, o = 0.0f;
    for (int v = 0; v < nw; ++v) m = fmaxf(m, wml[v][r][0]);
    for (int v = 0; v < nw; ++v) {
      const float f = wml[v][r][0] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(wml[v][r][0] - m);
      l = fmaf(f, wml[v][r][1], l);
      o = fmaf(f, wacc[v][r][d], o);
    }
    if (P.n_splits == 1) {
      if (d < P.io_hd) P.out[(row0 + r) * P.io_hd + d] = l == 0.0f ? 0.0f : o / l;
    } else {
      const int64_t pr = (row0 + r) * P.n_splits + split;
      P.part_acc[pr * T + d] = o;
      if (d == 0) reinterpret_cast<float2*>(P.part_ml)[pr] = make_float2(m, l);
    }
  }
}

// Joins the parts of a row: one wave a row, T / 64 dims a lane; lane v holds part v's
// maximum and sum, 64 parts a turn. Bound: launch and one round of loads, 2.3-4.5 us.
template <int T>
DEV void sparse_merge(const SparseParams& P) {
  constexpr int EPL = T / WAVE, UN = 8;
  const int lane = lane_id();
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / WAVE) + threadIdx.x / WAVE;
  if (row >= (int64_t)P.n_seqs * P.n_heads) return;
  const float2* ml = reinterpret_cast<const float2*>(P.part_ml) + row * P.n_splits;
  const float* acc = P.part_acc + row * P.n_splits * T + lane * EPL;
  float m = -kInf, l = 0.0f, o[EPL] = {};
  for (int v0 = 0; v0 < P.n_splits; v0 += WAVE) {
    const int nv = min(WAVE, P.n_splits - v0);
    const float2 x = ml[v0 + min(lane, nv - 1)];
    const float xm = lane < nv ? x.x : -kInf, top = fmaxf(m, wave_max(xm));
    const float f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);  // of the turns before
    const float part = xm == -kInf ? 0.0f : __builtin_amdgcn_exp2f(xm - top);
    m = top;
    l = l * f + wave_sum(part * x.y);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] *= f;
    for (int v = 0; v < nv; v += UN) {
      float a[UN][EPL];
#pragma unroll
      for (int i = 0; i < UN; ++i)
#pragma unroll
        for (int e = 0; e < EPL; ++e) a[i][e] = acc[(int64_t)(v0 + min(v + i, nv - 1)) * T + e];
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const float s = v + i < nv ? readlane_f(part, v + i) : 0.0f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[e] = fmaf(s, a[i][e], o[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e)
    if (lane * EPL + e < P.io_hd) P.out[row * P.io_hd + lane * EPL + e] = l == 0.0f ? 0.0f : o[e] / l;
}

}  // namespace

#define VK_KERNEL(NAME, THREADS, PARAMS, BODY) \
  extern "C" __global__ void __launch_bounds__(THREADS) NAME(const PARAMS P) { BODY; }

#define VK_INDEX(KV)                                                                   \
  VK_KERNEL(vk_index_update_kv##KV, kUpdateThreads, IndexUpdateParams, (index_update<KV, 128>(P)))  \
  VK_KERNEL(vk_index_update_kv##KV##_d64, kUpdateThreads, IndexUpdateParams, (index_update<KV, 64>(P)))
VK_INDEX(0) VK_INDEX(1) VK_INDEX(2) VK_INDEX(3)
VK_KERNEL(vk_index_read, 256, IndexReadParams, index_read(P))

#define VK_SELECT(TAG, QT, T, RT)                                                                       \
  VK_KERNEL(vk_page_select##TAG, kSelThreads, SelectParams, (page_select<QT, T, RT, false>(P)))          \
  VK_KERNEL(vk_page_select_rows##TAG, kSelThreads, SelectParams, (page_select<QT, T, RT, true>(P)))      \
  VK_KERNEL(vk_page_scores##TAG, kSelThreads, SelectParams, (page_scores<QT, T, RT>(P)))
#define VK_SELECT_Q(QT)                                                   \
  VK_SELECT(_r1_q##QT, QT, 128, 1) VK_SELECT(_r2_q##QT, QT, 128, 2)          \
  VK_SELECT(_d64_r1_q##QT, QT, 64, 1) VK_SELECT(_d64_r2_q##QT, QT, 64, 2)
VK_SELECT_Q(0) VK_SELECT_Q(1)
VK_KERNEL(vk_page_topk, 64 * kSelMaxWaves, SelectParams, page_topk<kSelMaxWaves>(P))

#define VK_SPARSE(KV, QT)                                                                                          \
  VK_KERNEL(vk_sparse_kv##KV##_r1_q##QT, 64 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 128, 1>(P)))         \
  VK_KERNEL(vk_sparse_kv##KV##_r2_q##QT, 32 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 128, 2>(P)))         \
  VK_KERNEL(vk_sparse_kv##KV##_d64_r1_q##QT, 64 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 64, 1>(P)))      \
  VK_KERNEL(vk_sparse_kv##KV##_d64_r2_q##QT, 32 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 64, 2>(P)))
#define VK_SPARSE_Q(KV) VK_SPARSE(KV, 0) VK_SPARSE(KV, 1)
VK_SPARSE_Q(0) VK_SPARSE_Q(1) VK_SPARSE_Q(2) VK_SPARSE_Q(3)
VK_KERNEL(vk_sparse_merge, 256, SparseParams, sparse_merge<128>(P))
VK_KERNEL(vk_sparse_merge_d64, 256, SparseParams, sparse_merge<64>(P))
