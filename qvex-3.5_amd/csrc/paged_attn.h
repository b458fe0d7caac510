// What the two forms of paged attention share (paged_attn.hip: calls of few rows;
// paged_chunk.hip: prompt chunks): their arguments, the steps from codes to
// bf16, the records of a split, the epilogue.
#pragma once
#include "paged.h"

namespace {

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pa_bf16x2 __attribute__((ext_vector_type(2)));
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));
typedef float pa_f32x2 __attribute__((ext_vector_type(2)));

constexpr int PA_ROWS = 16;            // rows of a tile of few rows
constexpr int PA_STEP = 128;           // keys that splits are multiples of
constexpr float PA_NONE = -3.0e38f;    // m before any visible key
constexpr float PA_SLACK = 8.0f;       // m moves when a score (base 2) passes it by more: P up to 256

struct PaArgs {
  KvPages c;
  KvRows r;
  const uint16_t* q;
  long q_token, q_head;
  const uint16_t* gate;
  long g_token, g_head;
  uint16_t* out;
  float* ws;                           // O [records][D], then (m, l) [records]
  size_t records;                      // [T * Hq][nsplit], or of shares [Hkv][shares + B][PA_ROWS]
  int Hq, kps, nsplit, vec, B, shares;
  float c2;                            // scale * log2(e): scores in base 2
};

__device__ __forceinline__ pa_bf16x8 as_pa8(const u32x4 v) { return __builtin_bit_cast(pa_bf16x8, v); }
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((pa_f32x2{lo, hi}), pa_bf16x2));
}
__device__ __forceinline__ float2* pa_ml(const PaArgs& a, int D) {
  return reinterpret_cast<float2*>(a.ws + a.records * D);
}

// A uniform word of the block table: a scalar load.
__device__ __forceinline__ int pa_page(const int32_t* t, int i) {
  return ((const __attribute__((address_space(4))) int32_t*)t)[i];
}

// A block's work: row tiles `tile`, `tile` + `tiles`, ... of kv head kh of sequence b. Workgroups go round
// the 8 XCDs and their engines in order of their number. Sequences of one length, grid
// [tiles * Hkv][B]: a sequence's tiles are neighbours, and read its keys at one time (us, 64 x 8 rows after 2000 bf16
// keys: 152; as below 170). With row offsets, sequences may leave blocks without rows, so blocks with
// rows must not lie a power of two apart: grid [B * Hkv][tiles], first tiles are neighbours, and each
// further row of the grid is rotated, so that the tiles of one sequence are too (us, int8 after 2000
// to 4000 keys, 64 sequences of one row, bound 64 | one of 512 rows and 63 of one | one of 512 and 15 of
// one, a sequence's tiles as neighbours 420 | 773 | 166, not rotated 102 | 327 | 527, rotated 106 | 223 | 189).
struct PaBlock {
  int b, kh, tile, tiles;
  __device__ __forceinline__ PaBlock(const PaArgs& a) {
    const uint32_t x = blockIdx.x, y = blockIdx.y, n = gridDim.x, heads = a.c.Hkv;
    uint32_t pair = x;
    if (a.r.cu) {
      const uint32_t turn = y == 0 ? 0 : y * ((64 + heads - n) & 63) % n;
      pair = x < turn ? x + n - turn : x - turn;
      b = pair / heads;
      tile = y;
      tiles = gridDim.y;
    } else {
      b = y;
      tile = x / heads;
      tiles = n / heads;
      pair = x - tile * heads;
    }
    kh = a.r.cu ? pair - b * heads : pair;
  }
};

// Shares: the 128-key steps of all sequences' first tiles, one after another, cut into `shares` equal runs, one
// per block of a kv head. Run i's part of sequence b leaves record i + b: every further part moves one of the two on.
__device__ __forceinline__ int pa_steps(const PaArgs& a, int b, int GQ) {
  const KvSeq s(a.r, b);
  const int keys = min(s.pos + min(s.n, (PA_ROWS - 1) / GQ + 1), a.r.width << a.c.shift);
  if (s.n == 0) return 0;
  // a sequence of more rows than a tile has a first step in any case: its block takes the other tiles too
  return max((max(keys, 0) + PA_STEP - 1) / PA_STEP, s.n * GQ > PA_ROWS ? 1 : 0);
}
__device__ __forceinline__ int pa_wave_sum(int x) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) x += __shfl_xor(x, m, 64);
  return __builtin_amdgcn_readfirstlane(x);
}

inline dim3 pa_grid(const PaArgs& a, int B, int tiles) {
  return a.r.cu ? dim3(a.c.Hkv * B, tiles, a.nsplit) : dim3(a.c.Hkv * tiles, B, a.nsplit);
}

__device__ __forceinline__ u32x4 pa_load8(const uint16_t* p, int vec) {
  if (vec) return load16(p);
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  return w;
}

// Codes e .. e + 7 of eight bytes as bf16.
template <int FMT>
__device__ __forceinline__ u32x4 codes8(uint32_t lo, uint32_t hi) {
  u32x4 o;
  if constexpr (FMT == QVEX_KV_FP8) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
    o[0] = pa_pack((float)(int8_t)lo, (float)(int8_t)(lo >> 8));
    o[1] = pa_pack((float)(int8_t)(lo >> 16), (float)(int8_t)(lo >> 24));
    o[2] = pa_pack((float)(int8_t)hi, (float)(int8_t)(hi >> 8));
    o[3] = pa_pack((float)(int8_t)(hi >> 16), (float)(int8_t)(hi >> 24));
  }
  return o;
}

// Codes 2 t and 2 t + 1 of two keys' words x, y: as bf16 pairs (x, y).
template <int FMT>
__device__ __forceinline__ void pair2(uint32_t x, uint32_t y, int t, uint32_t& a0, uint32_t& a1) {
  if constexpr (FMT == QVEX_KV_FP8) {
    const uint32_t w = __builtin_amdgcn_perm(y, x, t & 1 ? 0x07030602u : 0x05010400u);
    a0 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    a1 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
  } else {
    const int s = t & 1 ? 16 : 0;
    a0 = pa_pack((float)(int8_t)(x >> s), (float)(int8_t)(y >> s));
    a1 = pa_pack((float)(int8_t)(x >> (s + 8)), (float)(int8_t)(y >> (s + 8)));
  }
}

// The A operands of tiles 2 t and 2 t + 1: values 2 t and 2 t + 1 of each of eight keys' runs v.
template <int FMT, int VW>
__device__ __forceinline__ void gather2(const uint32_t (&v)[8][VW], int t, u32x4& a0, u32x4& a1) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (FMT == QVEX_KV_BF16) {
      a0[i] = __builtin_amdgcn_perm(v[2 * i + 1][t], v[2 * i][t], 0x05040100u);
      a1[i] = __builtin_amdgcn_perm(v[2 * i + 1][t], v[2 * i][t], 0x07060302u);
    } else {
      uint32_t x, y;
      pair2<FMT>(v[2 * i][t >> 1], v[2 * i + 1][t >> 1], t, x, y);
      a0[i] = x;
      a1[i] = y;
    }
  }
}

// The same of four keys.
template <int FMT, int VW>
__device__ __forceinline__ void gather2x4(const uint32_t (&v)[4][VW], int t, u32x2& a0, u32x2& a1) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (FMT == QVEX_KV_BF16) {
      a0[i] = __builtin_amdgcn_perm(v[2 * i + 1][t], v[2 * i][t], 0x05040100u);
      a1[i] = __builtin_amdgcn_perm(v[2 * i + 1][t], v[2 * i][t], 0x07060302u);
    } else {
      uint32_t x, y;
      pair2<FMT>(v[2 * i][t >> 1], v[2 * i + 1][t >> 1], t, x, y);
      a0[i] = x;
      a1[i] = y;
    }
  }
}

// Lane i of each 16-lane row, in every lane of that row.
template <int I>
__device__ __forceinline__ float row_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + I, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_lane_of(float v, int i) {   // i a constant after unrolling
  switch (i) {
    case 0: return row_lane<0>(v);
    case 1: return row_lane<1>(v);
    case 2: return row_lane<2>(v);
    case 3: return row_lane<3>(v);
    case 4: return row_lane<4>(v);
    case 5: return row_lane<5>(v);
    case 6: return row_lane<6>(v);
    case 7: return row_lane<7>(v);
    case 8: return row_lane<8>(v);
    case 9: return row_lane<9>(v);
    case 10: return row_lane<10>(v);
    case 11: return row_lane<11>(v);
    case 12: return row_lane<12>(v);
    case 13: return row_lane<13>(v);
    case 14: return row_lane<14>(v);
    default: return row_lane<15>(v);
  }
}

// The word with 0 for every infinity and NaN.
template <int FMT>
__device__ __forceinline__ uint32_t tame(uint32_t w) {
  if constexpr (FMT == QVEX_KV_BF16)
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
  uint32_t o = w;
  if constexpr (FMT == QVEX_KV_FP8) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((w >> (8 * i) & 0x7fu) == 0x7fu) o &= ~(0xffu << (8 * i));
  }
  return o;
}

// sigmoid(gate) of four dims of a row (1 without a gate), asked for where it is made, and the row's
// epilogue.
struct PaGate {
  uint16_t g[4];
  __device__ __forceinline__ PaGate(const PaArgs& a, int t, int h, int d) {
    if (!a.gate) return;
    const uint16_t* gp = a.gate + t * a.g_token + h * a.g_head + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = gp[i];
  }
  // seen: the row sees a key (one that does not is zero whatever its gate holds)
  __device__ __forceinline__ void store(const PaArgs& a, int t, int h, int d, int D, const float (&o)[4], bool seen) const {
    float f[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    if (a.gate && seen) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = 1.0f / (1.0f + expf(-bf16_to_f32(g[i])));
    }
    *reinterpret_cast<u32x2*>(a.out + ((size_t)t * a.Hq + h) * D + d) =
        u32x2{pack_bf16x2(o[0] * f[0], o[1] * f[1]), pack_bf16x2(o[2] * f[2], o[3] * f[3])};
  }
};

}  // namespace

namespace qvex {
// Launches the chunk form on checked arguments: `tiles` blocks of rows for the longest sequence.
constexpr int PA_CHUNK_ROWS = 128;
void paged_chunk_attention(const void* args, int format, int D, int tiles, int B, void* stream);
}  // namespace qvex
