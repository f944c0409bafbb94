// Device helpers shared by the gfx950 code objects: lane exchanges, conversions,
// tile loads through buffer descriptors and the misuse flag.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "velokv_params.h"

namespace {
using namespace velokv;

#define DEV static __device__ __forceinline__

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int BS = 16;    // tokens per block
constexpr int HD = 128;   // head_dim
constexpr int WAVE = 64;
constexpr float kNegInf = -__builtin_huge_valf();

template <typename T, typename F>
DEV T bitcast(F x) { return __builtin_bit_cast(T, x); }

DEV float h2f(uint16_t b) { return (float)bitcast<_Float16>(b); }
DEV uint16_t f2h(float x) { return bitcast<uint16_t>((_Float16)x); }  // IEEE RNE
DEV int lane_id() { return __lane_id(); }

// ---- cross-lane helpers (DPP inside a row of 16 lanes, ds_bpermute across rows)
template <int CTRL>
DEV float dpp(float x) {
  return bitcast<float>(__builtin_amdgcn_update_dpp(0, bitcast<int>(x), CTRL, 0xF, 0xF, false));
}
constexpr int DPP_QUAD_XOR1 = 0xB1;    // quad_perm [1,0,3,2]
constexpr int DPP_QUAD_XOR2 = 0x4E;    // quad_perm [2,3,0,1]
constexpr int DPP_ROW_ROR2 = 0x122;
constexpr int DPP_ROW_ROR4 = 0x124;
constexpr int DPP_ROW_ROR8 = 0x128;
constexpr int DPP_ROW_HALF_MIRROR = 0x141;
constexpr int DPP_ROW_MIRROR = 0x140;

DEV float shfl_xor(float x, int m) { return __shfl_xor(x, m, WAVE); }
// x of lane l ^ 32: v_permlane32_swap exchanges lanes 32..63 of its first
// operand with lanes 0..31 of its second (a VALU exchange, no LDS round trip);
// with both operands x, the second result holds x[l + 32] in lanes 0..31 and the
// first holds x[l - 32] in lanes 32..63.
DEV float xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(lane_id() < 32 ? r[1] : r[0]);
}

DEV float wave_max(float x) {
  x = fmaxf(x, dpp<DPP_QUAD_XOR1>(x));
  x = fmaxf(x, dpp<DPP_QUAD_XOR2>(x));
  x = fmaxf(x, dpp<DPP_ROW_HALF_MIRROR>(x));
  x = fmaxf(x, dpp<DPP_ROW_MIRROR>(x));
  x = fmaxf(x, shfl_xor(x, 16));
  x = fmaxf(x, shfl_xor(x, 32));
  return x;
}
DEV float wave_sum(float x) {
  x += dpp<DPP_QUAD_XOR1>(x);
  x += dpp<DPP_QUAD_XOR2>(x);
  x += dpp<DPP_ROW_HALF_MIRROR>(x);
  x += dpp<DPP_ROW_MIRROR>(x);
  x += shfl_xor(x, 16);
  x += shfl_xor(x, 32);
  return x;
}
// Reductions over the 16 lanes that share (lane & 3).
DEV float max_same_quadpos(float x) {
  x = fmaxf(x, dpp<DPP_ROW_ROR4>(x));
  x = fmaxf(x, dpp<DPP_ROW_ROR8>(x));
  x = fmaxf(x, shfl_xor(x, 16));
  x = fmaxf(x, shfl_xor(x, 32));
  return x;
}
DEV float sum_same_quadpos(float x) {
  x += dpp<DPP_ROW_ROR4>(x);
  x += dpp<DPP_ROW_ROR8>(x);
  x += shfl_xor(x, 16);
  x += shfl_xor(x, 32);
  return x;
}
DEV float readlane_f(float x, int l) { return bitcast<float>(__builtin_amdgcn_readlane(bitcast<int>(x), l)); }
DEV int readlane_i(int x, int l) { return __builtin_amdgcn_readlane(x, l); }

template <int CTRL>
DEV uint32_t dpp_u(uint32_t x, uint32_t old) { return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)x, CTRL, 0xF, 0xF, false); }
DEV uint32_t wave_max_u(uint32_t x) {
  x = max(x, dpp_u<DPP_QUAD_XOR1>(x, x));
  x = max(x, dpp_u<DPP_QUAD_XOR2>(x, x));
  x = max(x, dpp_u<DPP_ROW_HALF_MIRROR>(x, x));
  x = max(x, dpp_u<DPP_ROW_MIRROR>(x, x));
  return max(max((uint32_t)readlane_i((int)x, 0), (uint32_t)readlane_i((int)x, 16)),
             max((uint32_t)readlane_i((int)x, 32), (uint32_t)readlane_i((int)x, 48)));
}

// Sum over lanes 0 .. l.
DEV int wave_prefix_sum(int x) {
  x += (int)dpp_u<0x111>((uint32_t)x, 0);  // row_shr 1, 2, 4, 8
  x += (int)dpp_u<0x112>((uint32_t)x, 0);
  x += (int)dpp_u<0x114>((uint32_t)x, 0);
  x += (int)dpp_u<0x118>((uint32_t)x, 0);
  const int lane = lane_id(), a = readlane_i(x, 15), b = readlane_i(x, 31), c = readlane_i(x, 47);
  return x + (lane >= 16 ? a : 0) + (lane >= 32 ? b : 0) + (lane >= 48 ? c : 0);
}

// A float as an unsigned key of the same order (-0 as 0; not for NaN), and back.
DEV uint32_t order_key(float x) {
  const uint32_t u = bitcast<uint32_t>(x + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
DEV float key_value(uint32_t k) { return bitcast<float>((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }

// ---- int8 -> fp16 -----------------------------------------------------------
// Four signed int8 codes (little-endian bytes b0..b3) become two fp16 pairs that
// hold the codes exactly: (b0,b1) and (b2,b3). XOR 0x80 turns each byte into
// offset binary u = c + 128; v_perm_b32 places u under the exponent byte 0x64,
// which is the fp16 value 1024 + u; subtracting 1152 leaves c.
DEV void i8x4_to_h2x2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
  const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
  const half2v bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  lo = bitcast<uint32_t>(bitcast<half2v>(a) - bias);
  hi = bitcast<uint32_t>(bitcast<half2v>(b) - bias);
}
DEV float dot2(uint32_t a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2(bitcast<half2v>(a), bitcast<half2v>(b), c, false);
}
DEV float byte_to_f(uint32_t w, int byte) { return (float)(int8_t)((w >> (8 * byte)) & 0xFFu); }
DEV float half_lo(uint32_t w) { return h2f((uint16_t)(w & 0xFFFFu)); }
DEV float half_hi(uint32_t w) { return h2f((uint16_t)(w >> 16)); }
// Two fp32 values to an fp16 pair, each rounded to nearest even: one
// v_cvt_pk_f16_f32.
typedef float f32x2 __attribute__((ext_vector_type(2)));
DEV uint32_t pack_h2(float a, float b) {
  const f32x2 x = {a, b};
  return bitcast<uint32_t>(__builtin_convertvector(x, half2v));
}

template <int KV> struct Esz;
template <> struct Esz<KV_F32> { static constexpr int v = 4; };
template <> struct Esz<KV_F16> { static constexpr int v = 2; };
template <> struct Esz<KV_I8_REF> { static constexpr int v = 1; };
template <> struct Esz<KV_I8_BLK> { static constexpr int v = 1; };

// Per-lane vector of N dwords loaded with as few instructions as possible. K/V
// tiles are read exactly once per decode, so the loads are marked non-temporal.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int N> struct DW { uint32_t d[N]; };
template <int N>
DEV DW<N> load_dw(const uint8_t* p) {
  DW<N> r;
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i);
      r.d[4 * i] = v.x; r.d[4 * i + 1] = v.y; r.d[4 * i + 2] = v.z; r.d[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.d[0] = v.x; r.d[1] = v.y;
  } else {
    r.d[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}

// Misuse is reported, not trapped: the kernel or-s a flag into the context's
// error word (a vector atomic) and carries on with the clamped input.
DEV void flag_misuse(uint32_t* err, uint32_t bit) {
  if (err) __hip_atomic_fetch_or(err, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Buffer resource over one tile: base address and size in SGPRs, so the per-lane
// offset stays a fixed VGPR and address registers never alias load results.
// Word 3 = 0x00020000 (32-bit data format, the gfx9-family raw-buffer setting).
typedef __amdgpu_buffer_rsrc_t rsrc_t;
DEV rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  // the base is wave-uniform by construction; say so, so the descriptor lives in SGPRs
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  void* u = reinterpret_cast<void*>(((uint64_t)hi << 32) | lo);
  return __builtin_amdgcn_make_buffer_rsrc(u, 0, (int)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
// Cache policy of tile loads: V is streamed non-temporally. K rows are split
// over several load instructions (each covers a half (int8) or a quarter (fp16)
// of every 128-byte line of the tile), so K stays in the normal L2 policy unless
// its elements are bytes, where non-temporal measured faster.
constexpr int kAuxNT = 2;
template <int ESZ>
constexpr int k_aux() { return ESZ == 1 ? kAuxNT : 0; }
template <int N, int AUX = kAuxNT>
DEV DW<N> buf_load(rsrc_t r, uint32_t off) {
  DW<N> out;
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(off + 16 * i), 0, AUX);
      out.d[4 * i] = v.x; out.d[4 * i + 1] = v.y; out.d[4 * i + 2] = v.z; out.d[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, AUX);
    out.d[0] = v.x; out.d[1] = v.y;
  } else {
    out.d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, AUX);
  }
  return out;
}

}  // namespace
