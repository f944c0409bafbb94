// velokv_sparse.hip -- gfx950 kernels of sparse decode: the key index beside a
// pool, the choice of pages by it, and attention over the chosen pages.
//
// A code object of its own (velokv_sparse_gfx950.co), loaded beside the main one.
#include "velokv_device.h"

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

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
// A page with a key that is not finite has the scale infinity (it is chosen before
// any other).
// =============================================================================
template <int KV, int T>
DEV void index_update(const IndexUpdateParams& P) {
  constexpr int ESZ = Esz<KV>::v;
  constexpr int EPC = 16 / ESZ;                      // dims of a 16-byte chunk
  constexpr bool I8 = ESZ == 1;
  constexpr int LPT = I8 ? T / 32 : T / EPC;         // lanes that hold one token's chunks of a load
  constexpr int NI = 16 * T * ESZ / 1024;            // loads of 64 chunks per tile
  constexpr int NS = (I8 && T == 128) ? 2 : 1;       // sets of dims a lane holds
  constexpr int TLANES = (I8 && T == 64) ? 32 : 64;  // lanes l and l ^ 32 hold the same dims
  const int lane = lane_id();
  const int64_t unit = ((int64_t)P.wg0 + blockIdx.x) * (blockDim.x / WAVE) + threadIdx.x / WAVE;
  const int kvh = (int)(unit % P.n_kv_heads);
  const int64_t rest = unit / P.n_kv_heads;
  const int s = (int)(rest / P.max_pages);
  if (s >= P.n_seqs) return;
  const int ctx = max(0, min(P.context_lens[s], P.cap_tokens));
  const int first = P.first_tokens ? max(0, P.first_tokens[s]) : 0;
  const int ptok = 16 * P.page_tiles;
  const int64_t col = first / ptok + rest % P.max_pages;
  if (first >= ctx || col * ptok >= ctx) return;
  const int page = P.block_tables[(int64_t)table_row(P.seq_rows, s, P.bt_rows) * P.bt_stride + col];
  if (page < 0 || page >= P.n_pages) {
    if (lane == 0) flag_misuse(P.err, MISUSE_PAGE_OUT_OF_POOL);
    return;
  }
  const int nt = min(ptok, ctx - (int)col * ptok);
  const int tok = I8 ? (T == 128 ? lane >> 2 : (lane >> 1) & 15) : lane / LPT;  // of a load

  float lo[NS][EPC], hi[NS][EPC], bad = 0.0f;
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int e = 0; e < EPC; ++e) { lo[n][e] = kInf; hi[n][e] = -kInf; }
  for (int t = 0; t * BS < nt; ++t) {
    const int64_t tile = ((int64_t)page * P.page_tiles + t) * P.n_kv_heads + kvh;
    const uint8_t* base = P.kc + tile * P.tile_bytes;
    u32x4 c[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) c[j] = *reinterpret_cast<const u32x4*>(base + 1024 * j + 16 * lane);
    float scale = 1.0f;
    if constexpr (KV == KV_I8_BLK) scale = half_lo(*reinterpret_cast<const uint32_t*>(P.ks + tile * kBlkScaleStep));
    if constexpr (KV == KV_I8_REF) scale = reinterpret_cast<const float*>(P.ks + tile * P.stile_bytes)[tok];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n = NS == 2 ? j : 0;
      const int at = t * BS + (I8 ? tok : j * (WAVE / LPT) + tok);
      if (at < nt) {
#pragma unroll
        for (int e = 0; e < EPC; ++e) {
          float x;
          if constexpr (I8) x = byte_to_f(c[j][e / 4], e % 4) * scale;
          else if constexpr (KV == KV_F16) x = e % 2 ? half_hi(c[j][e / 2]) : half_lo(c[j][e / 2]);
          else x = bitcast<float>(c[j][e]);
          lo[n][e] = fminf(lo[n][e], x);
          hi[n][e] = fmaxf(hi[n][e], x);
          bad = fmaf(x, 0.0f, bad);
        }
      }
    }
  }
  // the lanes of one set of dims: all that differ in the token
  float top = 0.0f;
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int e = 0; e < EPC; ++e) {
#pragma unroll
      for (int m = LPT; m < TLANES; m *= 2) {
        lo[n][e] = fminf(lo[n][e], shfl_xor(lo[n][e], m));
        hi[n][e] = fmaxf(hi[n][e], shfl_xor(hi[n][e], m));
      }
      top = fmaxf(top, fmaxf(fabsf(lo[n][e]), fabsf(hi[n][e])));
    }
  top = wave_max(top);
  const bool ok = __builtin_amdgcn_ballot_w64(!(bad == 0.0f)) == 0;
  const float inv = ok ? code_scale(top) : 0.0f;
  const int64_t at = (int64_t)page * P.n_kv_heads + kvh;
  int8_t* codes = P.codes + at * 2 * T;
  // tokens 0's lanes write the lower bounds, tokens 1's the upper ones
  if (tok < 2) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int dim = I8 ? (T == 128 ? 32 * (lane & 3) + 16 * n : 32 * (lane & 1) + 16 * (lane >> 5)) : EPC * (lane % LPT);
      uint32_t w[EPC / 4];
#pragma unroll
      for (int e = 0; e < EPC; ++e) {
        const uint32_t b = (uint32_t)to_code(tok == 0 ? lo[n][e] : hi[n][e], inv) & 0xFFu;
        w[e / 4] = e % 4 ? w[e / 4] | b << (8 * (e % 4)) : b;
      }
      uint32_t* dst = reinterpret_cast<uint32_t*>(codes + tok * T + dim);
#pragma unroll
      for (int i = 0; i < EPC / 4; ++i) dst[i] = w[i];
    }
  }
  if (lane == 0) P.scales[at] = ok ? top / 127.0f : kInf;
}

// The bounds of listed pages as fp32: four dims a thread.
DEV void index_read(const IndexReadParams& P) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= P.n_chunks) return;
  const int per = P.io_hd / 4;
  const int64_t row = i / per;
  const int dim = (int)(i - row * per) * 4;
  const int kvh = (int)(row % P.n_kv_heads);
  const int page = P.pages[row / P.n_kv_heads];
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
// Selection. The bound of q . k over a page is sum_d max(q_d lo_d, q_d hi_d) =
// [min(q, 0), max(q, 0)] . [lo, hi], a product over 2 T dims; q and the bounds are
// int8 codes, so the sum is exact on v_mfma_i32_16x16x64_i8 (at most 128 x 127 x
// 127 < 2^24: exact in fp32 too) and the score
//     max over the group's heads of fp32(fp32(dot * page scale) * head scale)
// has the same bits however it is computed. Scores are kept as ordered 32-bit keys
// (larger key = chosen earlier); the pages that are always kept have the largest.
// =============================================================================
constexpr int kSelWaves = 4;
constexpr uint32_t kKeyKept = 0xFFFFFFFFu;


// Rows of the (sequence, KV head)'s queries as codes in LDS, negative parts first;
// rows past the group hold zeros. Returns after a barrier.
template <int QT, int T, int RT>
DEV void load_query_codes(const SelectParams& P, int s, int kvh, int8_t (*qc)[2 * T], float* qs) {
  const int lane = lane_id(), w = (int)threadIdx.x / WAVE, G = P.n_heads / P.n_kv_heads;
  constexpr int EPL = T / WAVE;
  for (int r = w; r < 16 * RT; r += kSelWaves) {
    float x[EPL], bad = 0.0f, top = 0.0f;
    const int64_t row = ((int64_t)s * P.n_heads + (int64_t)kvh * G + min(r, G - 1)) * P.io_hd;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int d = lane * EPL + e;
      x[e] = 0.0f;
      if (r < G && d < P.io_hd)
        x[e] = QT == DT_F32 ? reinterpret_cast<const float*>(P.q)[row + d] : h2f(reinterpret_cast<const uint16_t*>(P.q)[row + d]);
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

template <int QT, int T, int RT>
DEV void page_scores(const SelectParams& P) {
  constexpr int KJ = 2 * T / 64;  // products of 64 dims
  __shared__ __align__(16) int8_t qc[16 * RT][2 * T];
  __shared__ float qs[16 * RT];
  const int lane = lane_id(), n = lane & 15, g = lane >> 4, w = (int)threadIdx.x / WAVE;
  const int chunk = (int)(blockIdx.x % P.n_chunks);
  const int unit = (int)(blockIdx.x / P.n_chunks);
  const int kvh = unit % P.n_kv_heads, s = unit / P.n_kv_heads;
  const int G = P.n_heads / P.n_kv_heads;
  const int ctx = max(0, min(P.context_lens[s], P.cap_tokens));
  const int np = (ctx + P.page_tokens - 1) / P.page_tokens;
  if (np <= P.n_list) return;  // all pages are listed
  load_query_codes<QT, T, RT>(P, s, kvh, qc, qs);
  i32x4 qa[RT][KJ];
  float qsc[RT][4];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int j = 0; j < KJ; ++j) qa[rt][j] = *reinterpret_cast<const i32x4*>(&qc[16 * rt + n][64 * j + 16 * g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) qsc[rt][i] = qs[16 * rt + 4 * g + i];
  }
  const int32_t* bt = P.block_tables + (int64_t)table_row(P.seq_rows, s, P.bt_rows) * P.bt_stride;
  uint32_t* keys = P.keys + (int64_t)unit * P.max_pages;
  bool out = false;
  for (int p0 = (chunk * kSelWaves + w) * 16; p0 < np; p0 += P.n_chunks * kSelWaves * 16) {
    const int raw = bt[min(p0 + n, np - 1)];
    out |= raw < 0 || raw >= P.n_pool_pages;
    const int64_t at = (int64_t)min(max(raw, 0), P.n_pool_pages - 1) * P.n_kv_heads + kvh;
    const i32x4* c = reinterpret_cast<const i32x4*>(P.codes + at * 2 * T + 16 * g);
    i32x4 kb[KJ];
#pragma unroll
    for (int j = 0; j < KJ; ++j) kb[j] = c[4 * j];
    const float scale = P.scales[at];
    float best = -kInf;  // a score that is not a number counts as this
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      i32x4 dot = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KJ; ++j) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[rt][j], kb[j], dot, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = ((float)dot[i] * scale) * qsc[rt][i];
        if (16 * rt + 4 * g + i < G) best = fmaxf(best, x);
      }
    }
    best = fmaxf(best, shfl_xor(best, 16));
    best = fmaxf(best, shfl_xor(best, 32));
    const int page = p0 + n;
    uint32_t key = order_key(scale == kInf ? kInf : best);
    if (page < P.n_first || page >= np - P.n_last) key = kKeyKept;
    if (g == 0 && page < np) keys[page] = key;
  }
  if (__builtin_amdgcn_ballot_w64(out) != 0 && lane == 0) flag_misuse(P.err, MISUSE_PAGE_OUT_OF_POOL);
}

// The n_list pages with the largest keys, ties to the lower page, in ascending order.
// Radix selection: each round counts the next 8 bits of the keys that share the bits
// found so far and keeps the bin that holds the n_list-th largest; the last round
// leaves that key and how many of its equals belong to the list.
DEV void page_topk(const SelectParams& P) {
  __shared__ int hist[256];
  __shared__ int found[2];  // bin, keys still wanted in it
  __shared__ int wsum[2][kSelWaves];
  const int tid = (int)threadIdx.x, lane = lane_id(), w = tid / WAVE;
  const int unit = (int)blockIdx.x, s = unit / P.n_kv_heads;
  const int ctx = max(0, min(P.context_lens[s], P.cap_tokens));
  const int np = (ctx + P.page_tokens - 1) / P.page_tokens;
  int32_t* pages = P.pages + (int64_t)unit * P.n_list;
  if (np <= P.n_list) {
    for (int i = tid; i < P.n_list; i += 64 * kSelWaves) pages[i] = i < np ? i : -1;
    return;
  }
  const uint32_t* keys = P.keys + (int64_t)unit * P.max_pages;
  uint32_t prefix = 0;
  int want = P.n_list;
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < np; i += 64 * kSelWaves) {
      const uint32_t k = keys[i];
      if (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (w == 0) {  // bins 255 - 4 l - e of lane l, largest first
      int c[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) { c[e] = hist[255 - 4 * lane - e]; sum += c[e]; }
      int incl = sum;
      for (int m = 1; m < WAVE; m *= 2) {
        const int up = __shfl_up(incl, m, WAVE);
        if (lane >= m) incl += up;
      }
      int before = incl - sum;
      if (before < want && incl >= want) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (before < want && before + c[e] >= want) {
            found[0] = 255 - 4 * lane - e;
            found[1] = want - before;
            before = want;  // no later bin
          } else {
            before += c[e];
          }
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    want = found[1];
    __syncthreads();
  }
  // prefix is the n_list-th largest key: every larger one is listed, and the first `want` equal ones
  int above = 0, equal = 0;  // before this round's pages
  for (int p0 = 0; p0 < np; p0 += 64 * kSelWaves) {
    const int i = p0 + tid;
    const uint32_t k = i < np ? keys[i] : 0u;
    const uint64_t gt = __builtin_amdgcn_ballot_w64(i < np && k > prefix), eq = __builtin_amdgcn_ballot_w64(i < np && k == prefix);
    if (lane == 0) { wsum[0][w] = __builtin_popcountll(gt); wsum[1][w] = __builtin_popcountll(eq); }
    __syncthreads();
    int a = above, e = equal;
    for (int v = 0; v < kSelWaves; ++v) {
      if (v < w) { a += wsum[0][v]; e += wsum[1][v]; }
      above += wsum[0][v];
      equal += wsum[1][v];
    }
    const uint64_t below = (1ull << lane) - 1;
    a += __builtin_popcountll(gt & below);
    e += __builtin_popcountll(eq & below);
    if (i < np && (k > prefix || (k == prefix && e < want))) pages[a + min(e, want)] = i;
    __syncthreads();
  }
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

  if (w == 0) {  // the part's entries that name a page of the context
    const int32_t* bt = P.block_tables + (int64_t)table_row(P.seq_rows, s, P.bt_rows) * P.bt_stride;
    const int32_t* list = P.pages + (int64_t)unit * P.n_list;
    const int e1 = min(P.n_list, (split + 1) * P.split_entries), ptok = 16 * P.page_tiles;
    int count = 0;
    bool bad = false;
    for (int e0 = split * P.split_entries; e0 < e1; e0 += WAVE) {
      const int col = e0 + lane < e1 ? list[e0 + lane] : -1;
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
  __syncthreads();
  const int n_tiles = __builtin_amdgcn_readfirstlane(n_valid) * P.page_tiles;

  // q^T: row n of each 16-row tile, zeros past the group and past head_dim
  half8 qa[RT][F32 ? 1 : KC], qlo[RT][QSPLIT ? KC : 1];
  float qf[RT][F32 ? T / 4 : 1];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = 16 * rt + n;
    const int64_t off = (row0 + min(r, G - 1)) * P.io_hd;
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < T / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = 16 * j + 4 * g + e;
          float x = 0.0f;
          if (r < G && d < P.io_hd)
            x = QT == DT_F32 ? reinterpret_cast<const float*>(P.q)[off + d] : h2f(reinterpret_cast<const uint16_t*>(P.q)[off + d]);
          qf[rt][4 * j + e] = x;
        }
    } else {
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const int d = sparse_qdim<KV, T>(j, g);
        half8 x = {0, 0, 0, 0, 0, 0, 0, 0}, lo = x;
        if (r < G && d < P.io_hd) {
          if constexpr (QT == DT_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float v = reinterpret_cast<const float*>(P.q)[off + d + i];
              x[i] = (_Float16)v;
              lo[i] = (_Float16)(v - (float)x[i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = bitcast<_Float16>(reinterpret_cast<const uint16_t*>(P.q)[off + d + i]);
          }
        }
        qa[rt][j] = x;
        if constexpr (QSPLIT) qlo[rt][j] = lo;
      }
    }
  }

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
          float v = sc[i] * P.scale_log2, up = 0.0f;
          if constexpr (BLK) { v = sc[i] * st[u].ks[0] * P.scale_log2; up = __builtin_amdgcn_logf(fmaxf(st[u].vs[0], kMinScale)); }
          if constexpr (REF) { v = sc[i] * st[u].ks[i] * P.scale_log2; up = __builtin_amdgcn_logf(fmaxf(st[u].vs[i], kMinScale)); }
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

// Joins the parts of a row: one wave a row, T / 64 dims a lane.
template <int T>
DEV void sparse_merge(const SparseParams& P) {
  constexpr int EPL = T / WAVE;
  const int lane = lane_id();
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / WAVE) + threadIdx.x / WAVE;
  if (row >= (int64_t)P.n_seqs * P.n_heads) return;
  const float2* ml = reinterpret_cast<const float2*>(P.part_ml) + row * P.n_splits;
  const float* acc = P.part_acc + row * P.n_splits * T + lane * EPL;
  float m = -kInf, l = 0.0f, o[EPL] = {};
  for (int v = 0; v < P.n_splits; ++v) m = fmaxf(m, ml[v].x);
  for (int v = 0; v < P.n_splits; ++v) {
    const float2 x = ml[v];
    const float f = x.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(x.x - m);
    l = fmaf(f, x.y, l);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = fmaf(f, acc[(int64_t)v * T + e], o[e]);
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e)
    if (lane * EPL + e < P.io_hd) P.out[row * P.io_hd + lane * EPL + e] = l == 0.0f ? 0.0f : o[e] / l;
}

}  // namespace

#define VK_KERNEL(NAME, THREADS, PARAMS, BODY) \
  extern "C" __global__ void __launch_bounds__(THREADS) NAME(const PARAMS P) { BODY; }

#define VK_INDEX(KV)                                                                   \
  VK_KERNEL(vk_index_update_kv##KV, 256, IndexUpdateParams, (index_update<KV, 128>(P)))  \
  VK_KERNEL(vk_index_update_kv##KV##_d64, 256, IndexUpdateParams, (index_update<KV, 64>(P)))
VK_INDEX(0) VK_INDEX(1) VK_INDEX(2) VK_INDEX(3)
VK_KERNEL(vk_index_read, 256, IndexReadParams, index_read(P))

#define VK_SCORES(QT)                                                                              \
  VK_KERNEL(vk_page_scores_r1_q##QT, 64 * kSelWaves, SelectParams, (page_scores<QT, 128, 1>(P)))      \
  VK_KERNEL(vk_page_scores_r2_q##QT, 64 * kSelWaves, SelectParams, (page_scores<QT, 128, 2>(P)))      \
  VK_KERNEL(vk_page_scores_d64_r1_q##QT, 64 * kSelWaves, SelectParams, (page_scores<QT, 64, 1>(P)))   \
  VK_KERNEL(vk_page_scores_d64_r2_q##QT, 64 * kSelWaves, SelectParams, (page_scores<QT, 64, 2>(P)))
VK_SCORES(0) VK_SCORES(1)
VK_KERNEL(vk_page_topk, 64 * kSelWaves, SelectParams, page_topk(P))

#define VK_SPARSE(KV, QT)                                                                                          \
  VK_KERNEL(vk_sparse_kv##KV##_r1_q##QT, 64 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 128, 1>(P)))         \
  VK_KERNEL(vk_sparse_kv##KV##_r2_q##QT, 32 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 128, 2>(P)))         \
  VK_KERNEL(vk_sparse_kv##KV##_d64_r1_q##QT, 64 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 64, 1>(P)))      \
  VK_KERNEL(vk_sparse_kv##KV##_d64_r2_q##QT, 32 * kSparseMaxWaves, SparseParams, (sparse_attn<KV, QT, 64, 2>(P)))
#define VK_SPARSE_Q(KV) VK_SPARSE(KV, 0) VK_SPARSE(KV, 1)
VK_SPARSE_Q(0) VK_SPARSE_Q(1) VK_SPARSE_Q(2) VK_SPARSE_Q(3)
VK_KERNEL(vk_sparse_merge, 256, SparseParams, sparse_merge<128>(P))
VK_KERNEL(vk_sparse_merge_d64, 256, SparseParams, sparse_merge<64>(P))
