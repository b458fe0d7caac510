// Writing a paged KV cache and reading it back (KVCache.update and its fields,
// engine/model.py:149-176), in bf16 or quantized to 8 bits on the way in.
//
// A row is the D values of one position and kv head, and D / 8 lanes hold it, eight
// consecutive values each: one 16-byte load per lane, the row's largest magnitude
// by lane exchanges, one 8-byte store of codes (16 of bf16). A token's row is
// consecutive bytes of its page, so a single token writes whole 128-byte lines.
//
//   code = rne(x * (top / max|x|)),  scale = max|x| / top,  top = 127 or 448
//
// One scale per row: the attention can apply it to a whole score (K) or a whole
// weight (V), and codes of either format are exact in bf16. Magnitudes are compared
// as integers (the order of their bits), in which a NaN lies above every
// infinity and an infinity above every number.
//
// Large calls are bound by memory (a copy of 2 GiB reaches 4.9 TB/s here), small ones by
// their launch and one round trip, 2 to 3 us. Blocks go along a sequence's rows (x), then the
// sequences (y): neighbours write one sequence's pages (us, append of eight ragged sequences of up to
// 512 rows: 7.1; sequences side by side 8.0).
#include "paged.h"

namespace {

typedef float kv_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 kv_bf16x2 __attribute__((ext_vector_type(2)));

constexpr int KV_THREADS = 256;

// Eight consecutive bf16 as floats; vec: 16-byte aligned.
__device__ __forceinline__ void load8(const uint16_t* p, bool vec, float (&x)[8]) {
  if (vec) {
    const u32x4 w = load16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bf16_to_f32(p[i]);
  }
}

__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return w;
}

// Eight values of a row into slot `at` (LANES lanes hold the row, this one number lane of it).
template <int FMT, int LANES>
__device__ __forceinline__ void store_row(const float (&x)[8], long at, int lane, uint8_t* pages, float* scales) {
  constexpr int D = 8 * LANES;
  if constexpr (FMT == QVEX_KV_BF16) {
    if (at >= 0) *reinterpret_cast<u32x4*>(pages + at * (2 * D) + 16 * lane) = pack8(x);
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int m = 1; m < LANES; m *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
    if (at < 0) return;
    constexpr float TOP = FMT == QVEX_KV_INT8 ? 127.0f : 448.0f;
    const float a = __uint_as_float(top);
    const bool live = a >= 1e-30f && top < 0x7f800000u;
    const float inv = TOP / (live ? a : 1.0f);
    uint32_t w[2] = {0, 0};
    if constexpr (FMT == QVEX_KV_INT8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)(int)rintf(x[i] * inv) & 0xffu) << (8 * (i & 3));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, p, true);
      }
    }
    *reinterpret_cast<u32x2*>(pages + at * D + 8 * lane) = live ? u32x2{w[0], w[1]} : u32x2{0, 0};
    if (lane == 0) scales[at] = live ? a / TOP : top < 0x7f800000u ? 0.0f : __uint_as_float(0x7fc00000u);
  }
}

// Row w of a sequence's n * Hkv * 2: K and V of each (token, head). 16.8 MB in 7.1 us (2.4 TB/s; eight
// ragged sequences of up to 512 rows, 4 heads of 256, fp8), 3 us for a row of each of 64.
template <int FMT, int LANES>
__global__ __launch_bounds__(KV_THREADS) void paged_append_kernel(KvPages c, KvRows r, const uint16_t* __restrict__ k,
                                                                  long k_token, long k_head,
                                                                  const uint16_t* __restrict__ v, long v_token,
                                                                  long v_head, int vec) {
  constexpr int PER = KV_THREADS / LANES;
  const int b = blockIdx.y, lane = threadIdx.x % LANES;
  const KvSeq s(r, b);
  const long rows = (long)s.n * c.Hkv * 2;
  for (long w = (long)blockIdx.x * PER + threadIdx.x / LANES; w < rows; w += (long)gridDim.x * PER) {
    const bool isv = w & 1;
    const int h = (int)((w >> 1) % c.Hkv), i = (int)((w >> 1) / c.Hkv);
    const uint16_t* src = isv ? v + (s.first + i) * v_token + h * v_head : k + (s.first + i) * k_token + h * k_head;
    float x[8];
    load8(src + 8 * lane, vec, x);
    store_row<FMT, LANES>(x, kv_slot(c, r, b, h, s.pos + i), lane, isv ? c.v : c.k, isv ? c.vs : c.ks);
  }
}

// Rows of (token, head): Hq query heads, Hkv of K, Hkv of V; a block takes PER heads of
// one token, whose (cos, sin) its first rot / 2 threads evaluate once. 512 rows, 16 and 4 heads of 256, int8:
// 11.5 MB in 5.9 to 7.2 us, 4 rows 4.0: the projection's read, the norm's lane exchanges and the rotation
// through LDS follow each other, and a block has one round of them.
template <int FMT, int LANES>
__global__ __launch_bounds__(KV_THREADS) void paged_qk_rope_kernel(KvPages c, KvRows r,
                                                                   const uint16_t* __restrict__ proj, long p_stride,
                                                                   const uint16_t* __restrict__ q_norm,
                                                                   const uint16_t* __restrict__ k_norm, int Hq, int rot,
                                                                   const double* __restrict__ freqs, float eps,
                                                                   uint16_t* __restrict__ q_out, int vec) {
  constexpr int D = 8 * LANES, PER = KV_THREADS / LANES;
  __shared__ float2 turn[D / 2];
  __shared__ float rowbuf[PER][D];
  const int b = blockIdx.y, lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, half = rot / 2;
  const KvSeq s(r, b);
  const int heads = Hq + 2 * c.Hkv, groups = (heads + PER - 1) / PER;
  const double freq = (int)threadIdx.x < half ? freqs[threadIdx.x] : 0.0;
  for (long w = blockIdx.x; w < (long)s.n * groups; w += gridDim.x) {     // uniform over the block
    const int i = (int)(w / groups), h = (int)(w % groups) * PER + sub, p = s.pos + i;
    const bool used = h < heads, isq = h < Hq, isv = h >= Hq + c.Hkv;
    const int kh = isv ? h - Hq - c.Hkv : h - Hq;
    const uint16_t* src = proj + (s.first + i) * p_stride;
    src += isq ? (long)h * 2 * D : (long)Hq * 2 * D + (long)(h - Hq) * D;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (used) load8(src + 8 * lane, vec, x);
    float nw[8];
    load8((isq ? q_norm : k_norm) + 8 * lane, vec, nw);
    if ((int)threadIdx.x < half) {
      // revolutions in fp64, then an angle of at most half a turn in fp32
      double turns = (double)p * freq * 0.15915494309189533577;
      turns -= rint(turns);
      float sn, cs;
      sincosf((float)(turns * 6.283185307179586477), &sn, &cs);
      turn[threadIdx.x] = make_float2(cs, sn);
    }
    if (used && !isv) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
      for (int m = 1; m < LANES; m *= 2) ss += __shfl_xor(ss, m, 64);
      const float inv = rsqrtf(ss / (float)D + eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= inv * nw[e];
        rowbuf[sub][8 * lane + e] = x[e];
      }
    }
    __syncthreads();
    if (used && !isv && 8 * lane < rot) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * lane + e;
        if (d < half) {
          const float2 t = turn[d];
          x[e] = x[e] * t.x - rowbuf[sub][d + half] * t.y;
        } else if (d < rot) {
          const float2 t = turn[d - half];
          x[e] = x[e] * t.x + rowbuf[sub][d - half] * t.y;
        }
      }
    }
    if (used && isq) {
      *reinterpret_cast<u32x4*>(q_out + ((long)(s.first + i) * Hq + h) * D + 8 * lane) = pack8(x);
    } else if (used) {
      store_row<FMT, LANES>(x, kv_slot(c, r, b, kh, p), lane, isv ? c.v : c.k, isv ? c.vs : c.ks);
    }
    __syncthreads();
  }
}

__device__ __forceinline__ void unpack8(int fmt, const u32x4 w, float (&x)[8]) {
  if (fmt == QVEX_KV_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  } else if (fmt == QVEX_KV_INT8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3)));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const kv_f32x2 f = i & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i >> 1], true)
                               : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i >> 1], false);
      x[2 * i] = f[0];
      x[2 * i + 1] = f[1];
    }
  }
}

// 4 x 8192 rows of 4 heads of 256 from int8 to bf16: 202 MB in 47 us, 4.3 TB/s.
template <int FMT, int LANES, typename OUT>
__global__ __launch_bounds__(KV_THREADS) void paged_read_kernel(KvPages c, KvRows r, OUT* __restrict__ k_out,
                                                                OUT* __restrict__ v_out) {
  constexpr int D = 8 * LANES, PER = KV_THREADS / LANES, ROW = D * kv_bytes(FMT);
  const int b = blockIdx.y, lane = threadIdx.x % LANES;
  const KvSeq s(r, b);
  const long rows = (long)s.n * c.Hkv * 2;
  for (long w = (long)blockIdx.x * PER + threadIdx.x / LANES; w < rows; w += (long)gridDim.x * PER) {
    const bool isv = w & 1;
    const int h = (int)((w >> 1) % c.Hkv), i = (int)((w >> 1) / c.Hkv);
    const long at = kv_slot(c, r, b, h, s.pos + i);
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (at >= 0) {
      const uint8_t* src = (isv ? c.v : c.k) + at * ROW + lane * (ROW / LANES);
      u32x4 raw = {0, 0, 0, 0};
      if constexpr (FMT == QVEX_KV_BF16) {
        raw = load16(src);
      } else {
        const u32x2 half = *reinterpret_cast<const u32x2*>(src);
        raw[0] = half[0];
        raw[1] = half[1];
      }
      unpack8(FMT, raw, x);
      if constexpr (FMT != QVEX_KV_BF16) {
        const float sc = (isv ? c.vs : c.ks)[at];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= sc;
      }
    }
    OUT* dst = (isv ? v_out : k_out) + ((long)(s.first + i) * c.Hkv + h) * D + 8 * lane;
    if constexpr (sizeof(OUT) == 2) {
      *reinterpret_cast<u32x4*>(dst) = pack8(x);
    } else {
      *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
  }
}

// Blocks along a sequence's rows: what L rows need, at most 4 rounds of the chip over all sequences.
unsigned kv_grid(long blocks, int B) {
  const long most = (8192 + B - 1) / B;
  return (unsigned)(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

}  // namespace

#define KV_DISPATCH(fn_, fmt, D, grid, st, ...)                                                          \
  do {                                                                                                   \
    if ((fmt) == QVEX_KV_BF16 && (D) == 256) hipLaunchKernelGGL((fn_<QVEX_KV_BF16, 32>), grid, dim3(KV_THREADS), 0, st, __VA_ARGS__); \
    else if ((fmt) == QVEX_KV_BF16) hipLaunchKernelGGL((fn_<QVEX_KV_BF16, 16>), grid, dim3(KV_THREADS), 0, st, __VA_ARGS__);          \
    else if ((fmt) == QVEX_KV_INT8 && (D) == 256) hipLaunchKernelGGL((fn_<QVEX_KV_INT8, 32>), grid, dim3(KV_THREADS), 0, st, __VA_ARGS__); \
    else if ((fmt) == QVEX_KV_INT8) hipLaunchKernelGGL((fn_<QVEX_KV_INT8, 16>), grid, dim3(KV_THREADS), 0, st, __VA_ARGS__);          \
    else if ((D) == 256) hipLaunchKernelGGL((fn_<QVEX_KV_FP8, 32>), grid, dim3(KV_THREADS), 0, st, __VA_ARGS__);                      \
    else hipLaunchKernelGGL((fn_<QVEX_KV_FP8, 16>), grid, dim3(KV_THREADS), 0, st, __VA_ARGS__);                                      \
  } while (0)

extern "C" int qvex_paged_append(const qvex_kv_pages* pages, const qvex_kv_rows* rows, const uint16_t* k, long k_token,
                                 long k_head, const uint16_t* v, long v_token, long v_head, void* stream) {
  const char* fn = "qvex_paged_append";
  KvPages c;
  KvRows r;
  if (const int rc = kv_check(fn, pages, rows, &c, &r)) return rc;
  if (r.T == 0) return QVEX_OK;
  QVEX_CHECK_ARG(k && v && qvex_aligned(k, 2) && qvex_aligned(v, 2), "%s: null or misaligned k or v", fn);
  const int vec = (k_token % 8 | k_head % 8 | v_token % 8 | v_head % 8) == 0 && qvex_aligned(k, 16) && qvex_aligned(v, 16);
  const int per = KV_THREADS / (pages->D / 8);
  const dim3 grid(kv_grid(((long)r.L * c.Hkv * 2 + per - 1) / per, rows->B), rows->B);
  KV_DISPATCH(paged_append_kernel, pages->format, pages->D, grid, (hipStream_t)stream, c, r, k, k_token, k_head, v,
              v_token, v_head, vec);
  QVEX_CHECK_LAUNCH(fn);
  return QVEX_OK;
}

extern "C" int qvex_paged_qk_rope(const qvex_kv_pages* pages, const qvex_kv_rows* rows, const uint16_t* proj,
                                  long p_stride, const uint16_t* q_norm, const uint16_t* k_norm, int Hq, int rot_dim,
                                  const double* freqs, float eps, uint16_t* q_out, void* stream) {
  const char* fn = "qvex_paged_qk_rope";
  KvPages c;
  KvRows r;
  if (const int rc = kv_check(fn, pages, rows, &c, &r)) return rc;
  const int D = pages->D;
  QVEX_CHECK_ARG(Hq >= 1 && Hq <= 16384 && Hq % c.Hkv == 0, "%s: Hq=%d Hkv=%d", fn, Hq, c.Hkv);
  QVEX_CHECK_ARG(rot_dim >= 0 && rot_dim <= D && rot_dim % 2 == 0, "%s: rot_dim=%d must be even, 0..D=%d", fn, rot_dim,
                 D);
  QVEX_CHECK_ARG(p_stride >= (long)Hq * 2 * D + 2L * c.Hkv * D, "%s: p_stride=%ld too small", fn, p_stride);
  if (r.T == 0) return QVEX_OK;
  QVEX_CHECK_ARG(proj && q_norm && k_norm && q_out && (freqs || rot_dim == 0), "%s: null pointer", fn);
  QVEX_CHECK_ARG(qvex_aligned(proj, 2) && qvex_aligned(q_norm, 2) && qvex_aligned(k_norm, 2) &&
                     qvex_aligned(q_out, 16) && qvex_aligned(freqs, 8),
                 "%s: q_out must be 16-byte aligned, freqs 8-byte", fn);
  const int vec = p_stride % 8 == 0 && qvex_aligned(proj, 16) && qvex_aligned(q_norm, 16) && qvex_aligned(k_norm, 16);
  const int per = KV_THREADS / (D / 8);
  const dim3 grid(kv_grid((long)r.L * ((Hq + 2 * c.Hkv + per - 1) / per), rows->B), rows->B);
  KV_DISPATCH(paged_qk_rope_kernel, pages->format, D, grid, (hipStream_t)stream, c, r, proj, p_stride, q_norm, k_norm,
              Hq, rot_dim, freqs, eps, q_out, vec);
  QVEX_CHECK_LAUNCH(fn);
  return QVEX_OK;
}

namespace {
template <int FMT, int LANES>
void launch_read(dim3 grid, hipStream_t st, const KvPages& c, const KvRows& r, void* k, void* v, int f32) {
  if (f32)
    hipLaunchKernelGGL((paged_read_kernel<FMT, LANES, float>), grid, dim3(KV_THREADS), 0, st, c, r, (float*)k, (float*)v);
  else
    hipLaunchKernelGGL((paged_read_kernel<FMT, LANES, uint16_t>), grid, dim3(KV_THREADS), 0, st, c, r, (uint16_t*)k,
                       (uint16_t*)v);
}
}  // namespace

extern "C" int qvex_paged_read(const qvex_kv_pages* pages, const qvex_kv_rows* rows, void* k_out, void* v_out,
                               int out_f32, void* stream) {
  const char* fn = "qvex_paged_read";
  KvPages c;
  KvRows r;
  if (const int rc = kv_check(fn, pages, rows, &c, &r)) return rc;
  if (r.T == 0) return QVEX_OK;
  QVEX_CHECK_ARG(k_out && v_out && qvex_aligned(k_out, 16) && qvex_aligned(v_out, 16),
                 "%s: the outputs must be 16-byte aligned, not null", fn);
  const int per = KV_THREADS / (pages->D / 8);
  const dim3 grid(kv_grid(((long)r.L * c.Hkv * 2 + per - 1) / per, rows->B), rows->B);
  const auto go = pages->D == 256 ? (pages->format == QVEX_KV_BF16   ? &launch_read<QVEX_KV_BF16, 32>
                                     : pages->format == QVEX_KV_INT8 ? &launch_read<QVEX_KV_INT8, 32>
                                                                     : &launch_read<QVEX_KV_FP8, 32>)
                                  : (pages->format == QVEX_KV_BF16   ? &launch_read<QVEX_KV_BF16, 16>
                                     : pages->format == QVEX_KV_INT8 ? &launch_read<QVEX_KV_INT8, 16>
                                                                     : &launch_read<QVEX_KV_FP8, 16>);
  go(grid, (hipStream_t)stream, c, r, k_out, v_out, out_f32);
  QVEX_CHECK_LAUNCH(fn);
  return QVEX_OK;
}
