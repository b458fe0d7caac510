// Paged attention of prompt chunks: paged_attn.hip's sums for calls of many rows.
//
// A block is 128 rows of one kv head (32 per wave, so that an operand from LDS
// serves two 16-row tiles), and 64 keys at a time go from the pages through
// registers, where codes become bf16, into LDS, double-buffered:
//   S^T[keys x rows] = K Q^T and O^T[dims x rows] += V^T P^T with 32x32x16 products. Lane
//   (hf, li) = (lane / 32, lane % 32) ends with scores of q row li and keys
//   8 (i / 4) + 4 hf + i % 4 of each 32 (i < 16); eight of them, as bf16, are its B operand
//   of a 16-key step of the second product, whose A operand holds the same eight
//   keys of one dim: V is stored in LDS by dims, its keys in that order.
// LDS, in 16-byte units: K's row r holds unit c at c ^ (r % 16); V's row of dim d is
// row d with its low two bits XORed by d / 16 % 4, unit c at c ^ (d / 4 % 4) ^ (d / 64): the 16
// lanes of one pass of a read hit 16 different bank groups. Writes do not always: V's 8-byte halves cost 258 cycles of
// conflicts a step, codes of K (a lane's 16 are two units, so a pass hits every other unit of a row) 255.
// A lane's 16 keys of a tile are one scale each for all its rows: a 16-lane row of
// the wave holds them, and a product takes scale i by DPP broadcast.
// Scores, m, l, O and the two bf16 terms of P as in paged_attn.hip: the output's error is its own rounding's (1.66e-3 of
// its norm; with one term 2.34e-3). Both terms' products take one operand of V from LDS, and the terms are
// made beside the products before, so the second costs the matrix cores' time (us, one term | two: after 16384 keys
// int8 185 | 215, bf16 165 | 198, fp8 171 | 194, after 3584 bf16 61 | 69, merge included).
//
// 16 query and 4 kv heads of 256: 512 positions after 3584 bf16 keys 63 to 66 us and 8.8 of merging, after 16384
// int8 keys 204 to 210 and 8.5 (670 TFLOP/s, the second term's products not counted). One wave per SIMD holds
// 32 rows of Q and O in 192 registers. By the counters a step of 64 int8 keys takes 6,850 cycles: in 60 % of them the
// wave issues (96 products, 700 other vector, 150 LDS instructions, 4 cycles each), in 19 % it waits for a matrix core
// that is busy (44 % of the time), in 21 % for LDS (active 30 %), memory or the barrier. No one of them bounds it alone: what stands
// beside no product, the scores' scales, maxima and vote, a lone wave cannot hide. Two waves per SIMD that share 32 rows (each one key
// tile's scores, half the dims of O, weights exchanged in LDS) measured, with one term, us, int8 | bf16 after
// 16384 keys | bf16 after 3584: 171 | 168 | 65 against 185 | 171 | 62 (merge included). A taken branch costs a lone
// wave some 200 cycles (rescaling O under a branch per tile of it 294 us against 189), so what is rare lies behind the
// loop (fp8 187 -> 180).
#include "paged_attn.h"

namespace {

typedef float pc_f32x16 __attribute__((ext_vector_type(16)));

constexpr int PC_KEYS = 64;            // keys per step
constexpr int PC_AHEAD = 8;            // operands of the second-next products asked for ahead

template <int I = 0>
__device__ __forceinline__ void scale16(pc_f32x16& s, float v) {
  if constexpr (I < 16) {
    s[I] *= row_lane<I>(v);
    scale16<I + 1>(s, v);
  }
}

// Value x of four that are the same for the wave (an array would be indexed in memory).
__device__ __forceinline__ uint32_t pick(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, int x) {
  const uint32_t lo = x & 1 ? a1 : a0, hi = x & 1 ? a3 : a2;
  return x & 2 ? hi : lo;
}

template <int FMT, int D>
__global__ __launch_bounds__(256, 1) void paged_chunk_kernel(PaArgs a) {
#pragma clang fp contract(off)
  constexpr int EB = kv_bytes(FMT), ROW = D * EB, KS = D / 16, NT = D / 32;
  constexpr int KU = PC_KEYS * ROW / 4096;       // 16-byte loads of K per thread and step
  constexpr int LPR = ROW / 16, KSTEP = 256 / LPR;   // lanes per key row, keys per load of the block
  constexpr int E = D / 16, VW = E * EB / 4;     // a thread's part of V and step: E dims (VW words) of four keys
  constexpr int K_BYTES = PC_KEYS * D * 2, STAGE = 2 * K_BYTES;
  // the product of V that the next step's V starts beside: any, or (fewer products to spread it over) the second tile's
  // (us after 16384 keys, the first | the second tile's: 256-dim heads int8 214 | 215, bf16 200 | 203, fp8 198 | 202,
  // 128-dim heads 250 | 250, 217 | 217, 240 | 233)
  constexpr int V_FIRST = D == 256 ? 0 : 2 * NT;
  __shared__ __align__(1024) uint8_t lds[2 * STAGE];
  __shared__ uint32_t blank[4];                  // rows of each wave that see nothing
  __shared__ int odd;                            // some V has a NaN or an infinity that not all rows see
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int li = lane & 31, hf = lane >> 5;
  const PaBlock blk(a);
  const int b = blk.b, kh = blk.kh, split = blockIdx.z, GQ = a.Hq / a.c.Hkv;
  const KvSeq s(a.r, b);
  const int cap = a.r.width << a.c.shift, rows = s.n * GQ, mask = (1 << a.c.shift) - 1;
  const int32_t* table = a.r.table + b * a.r.stride;
  const int k_lo = split * a.kps;

  for (int tile = blk.tile; tile * qvex::PA_CHUNK_ROWS < rows; tile += blk.tiles) {
    const int r0 = tile * qvex::PA_CHUNK_ROWS;
    const int last = min(rows, r0 + qvex::PA_CHUNK_ROWS) - 1;
    const int keys = min(s.pos + last / GQ + 1, cap);             // that any row of the block sees
    const int k_hi = split == a.nsplit - 1 ? keys : min(k_lo + a.kps, keys);
    if (k_lo >= k_hi) continue;                                   // uniform; the merge does not read it
    const int first_lim = s.pos + r0 / GQ;                        // last key of the block's first row
    const int w0 = r0 + 32 * wave, row = w0 + li;
    const bool used = row < rows;
    const int i = used ? row / GQ : 0, g = used ? row - i * GQ : 0;
    const int rlim = used ? min(s.pos + i, cap - 1) : -1;
    const int w_lim = s.pos + w0 / GQ;                            // of the wave's first row
    const int k_last = k_lo + (k_hi - 1 - k_lo) / PC_KEYS * PC_KEYS;   // the last step, fetched again behind it

    u32x4 qa[KS];
    const uint16_t* qp = a.q + (s.first + i) * a.q_token + (kh * GQ + g) * a.q_head + 8 * hf;
#pragma unroll
    for (int st = 0; st < KS; ++st) qa[st] = used ? pa_load8(qp + 16 * st, a.vec) : u32x4{0, 0, 0, 0};

    // ---- a step's keys: pages to registers, registers to LDS
    u32x4 kraw[KU];
    uint32_t vraw[4][VW];
    float ksn[2], vsn[2];
    uint32_t s0, s1, s2, s3;                                      // first slots of a step's 16-key groups
    // Lane x finds group x % 4: one load a step before and 20 instructions (us after 16384 keys, int8, 256- | 128-dim
    // heads: 181 | 219; as scalar code, 80 instructions, 187 | 228)
    const int x16 = 16 * (lane & 3);
    int asked;                                                    // the page of the next step's group
    auto ask = [&](int kb) __attribute__((always_inline)) { asked = table[min((kb + x16) >> a.c.shift, a.r.width - 1)]; };
    auto locate = [&](int kb) __attribute__((always_inline)) {    // returns which of the pages there are
      const bool ok = asked >= 0 && asked < a.c.n_pages;
      const uint32_t at = (((uint32_t)(ok ? asked : 0) * a.c.Hkv + kh) << a.c.shift) + ((kb + x16) & mask);
      s0 = __builtin_amdgcn_readlane(at, 0);
      s1 = __builtin_amdgcn_readlane(at, 1);
      s2 = __builtin_amdgcn_readlane(at, 2);
      s3 = __builtin_amdgcn_readlane(at, 3);
      ask(min(kb + PC_KEYS, k_last));
      return (int)__ballot(ok) & 15;
    };
    // a lane's scale of key tile kt: key 8 (x / 4) + 4 hf + x % 4 of it, x = lane % 16
    const uint32_t sc_at = 8 * ((lane >> 2) & 1) + 4 * hf + (lane & 3);
    auto scale_of = [&](const float* p, int kt) __attribute__((always_inline)) {
      return p[(lane & 8 ? (kt ? s3 : s1) : (kt ? s2 : s0)) + sc_at];
    };
    auto fetch_k = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < KU; ++u) {                              // KSTEP / 4 keys of one 16-key group per wave
        const int key = KSTEP * u + (KSTEP / 4) * wave + lane / LPR;
        const uint8_t* base = a.c.k + (uint64_t)pick(s0, s1, s2, s3, (KSTEP * u + (KSTEP / 4) * wave) >> 4) * ROW;
        kraw[u] = load16(base + (uint32_t)((key & 15) * ROW + 16 * (lane % LPR)));
      }
      if constexpr (EB == 1) {
        ksn[0] = scale_of(a.c.ks, 0);
        ksn[1] = scale_of(a.c.ks, 1);
      }
    };
    const int vq = lane >> 4, vc = lane & 15;                     // keys 4 vq .. + 3 of the wave's 16, dims E vc .. + E - 1
    auto fetch_v = [&]() __attribute__((always_inline)) {
      const uint8_t* base = a.c.v + (uint64_t)pick(s0, s1, s2, s3, wave) * ROW;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint8_t* p = base + (uint32_t)((4 * vq + e) * ROW + 4 * VW * vc);
        if constexpr (VW == 2) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(p);
          vraw[e][0] = w[0];
          vraw[e][1] = w[1];
        } else {
#pragma unroll
          for (int u = 0; u < VW / 4; ++u) {
            const u32x4 w = load16(p + 16 * u);
#pragma unroll
            for (int x = 0; x < 4; ++x) vraw[e][4 * u + x] = w[x];
          }
        }
      }
      if constexpr (EB == 1) {
        vsn[0] = scale_of(a.c.vs, 0);
        vsn[1] = scale_of(a.c.vs, 1);
      }
    };
    // Before a step goes to LDS: what no row of the block sees is not data, and its values (and their scales)
    // become 0, since 0 times a NaN is none. So does a NaN or an infinity that some rows do not see: the
    // rows that do are marked at the end.
    auto clean = [&](int kb, int ok_all) __attribute__((always_inline)) {
      if (__builtin_expect(kb + PC_KEYS <= min(first_lim + 1, k_hi) && ok_all == 15, 1)) return;
      bool any = false;
      if constexpr (EB == 1) {
        const int x = lane & 15;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const int kk = 32 * kt + 8 * (x >> 2) + 4 * hf + (x & 3);
          const bool live = kb + kk < k_hi && ok_all >> (kk >> 4) & 1;
          const bool wild = live && kb + kk > first_lim && !(fabsf(vsn[kt]) < INFINITY);
          if (!live || wild) vsn[kt] = 0.0f;
          any |= wild;
        }
      }
      if constexpr (FMT != QVEX_KV_INT8) {
        const bool v_ok = ok_all >> wave & 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = kb + 16 * wave + 4 * vq + e;
#pragma unroll
          for (int u = 0; u < VW; ++u) {
            const uint32_t w = key >= k_hi || !v_ok ? 0 : vraw[e][u], w1 = key > first_lim ? tame<FMT>(w) : w;
            any |= w1 != w;
            vraw[e][u] = w1;
          }
        }
      }
      if (__builtin_expect(any, 0)) odd = 1;
    };
    // Pieces of a step's way to LDS, K's and V's
    constexpr int KP = EB == 2 ? KU : 2 * KU, VP = E / 2;
    const int kw_at = ((KSTEP / 4) * wave + lane / LPR) * (2 * D);
    auto stage_k = [&](int to, int x) __attribute__((always_inline)) {
      const int u = EB == 2 ? x : x / 2, h = x & 1;
      const int key = (KSTEP * u + (KSTEP / 4) * wave + lane / LPR) & 15, c = lane % LPR;
      uint8_t* kr = lds + (to ^ kw_at) + KSTEP * u * (2 * D);
      if constexpr (EB == 2) {
        *reinterpret_cast<u32x4*>(kr + ((c ^ key) << 4)) = kraw[u];
      } else {
        *reinterpret_cast<u32x4*>(kr + (((2 * c + h) ^ key) << 4)) = codes8<FMT>(kraw[u][2 * h], kraw[u][2 * h + 1]);
      }
    };
    // dims E vc + 2 x, + 1: four keys of each, a half of unit 2 (wave % 2) + vq % 2
    const int vw_at = K_BYTES + (wave >> 1) * (D * 64) + 64 * E * vc + 8 * (vq >> 1);
    auto stage_v = [&](int to, int x) __attribute__((always_inline)) {
      u32x2 b0, b1;
      gather2x4<FMT, VW>(vraw, x, b0, b1);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int n = 2 * x + y;
        const int r = (n & 3) ^ (E == 16 ? vc & 3 : (vc >> 1) & 3);
        const int f = E == 16 ? ((n >> 2) ^ (vc >> 2)) & 3 : ((2 * vc + (n >> 2)) ^ (vc >> 3)) & 3;
        *reinterpret_cast<u32x2*>(lds + (to ^ vw_at) + (n & ~3) * 64 + r * 64 + (((2 * (wave & 1) + (vq & 1)) ^ f) << 4)) =
            y ? b1 : b0;
      }
    };

    // ---- operands from LDS: K's of both key tiles, then V's. The lane's addresses are kept, the buffer's bit flipped
    int k_at[KS < 8 ? KS : 8], v_at[2][4];                        // K: step st at entry st % 8, + 256 from 8
#pragma unroll
    for (int st = 0; st < KS && st < 8; ++st) k_at[st] = li * (2 * D) + (((2 * st + hf) ^ (li & 15)) << 4);
#pragma unroll
    for (int x = 0; x < 2; ++x)                                   // V: even and odd dim tiles; 2 t ^ (n / 2)
#pragma unroll
      for (int y = 0; y < 4; ++y)
        v_at[x][y] = K_BYTES + ((32 * x + (li & ~3)) | ((li & 3) ^ ((2 * x + (li >> 4)) & 3))) * 64 +
                     ((hf ^ y ^ ((li >> 2) & 3)) << 4);
    auto operand = [&](int x) __attribute__((always_inline)) {
      if (x < 2 * KS) {
        const int kt = x / KS, st = x % KS;
        return load16(lds + k_at[st % 8] + (kt * 64 * D + (st >> 3) * 256));
      }
      const int y = x - 2 * KS, kt = y / (2 * NT), t = y / NT % 2, n = y % NT;
      return load16(lds + v_at[n & 1][(2 * t) ^ ((n >> 1) & 3)] + (kt * (D * 64) + (n >> 1) * 4096));
    };

    const pc_f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    float m = PA_NONE, l = 0.0f;
    pc_f32x16 o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = zero;

    // step j + 1 goes to LDS beside the products of step j, from registers that were loaded during step j - 1
    if (threadIdx.x == 0) odd = 0;
    __syncthreads();
    ask(k_lo);
    int ok = locate(k_lo);
    fetch_k();
    fetch_v();
    float ksc[2] = {ksn[0], ksn[1]}, vsc[2];
    clean(k_lo, ok);
    vsc[0] = vsn[0];
    vsc[1] = vsn[1];
#pragma unroll
    for (int x = 0; x < KP; ++x) stage_k(0, x);
#pragma unroll
    for (int x = 0; x < VP; ++x) stage_v(0, x);
    int ok_next = locate(min(k_lo + PC_KEYS, k_last));
    fetch_k();
    fetch_v();
    __syncthreads();
    int to = STAGE;
#pragma unroll 1
    for (int kb = k_lo; kb < k_hi; kb += PC_KEYS, to ^= STAGE) {
      const int ok_further = locate(min(kb + 2 * PC_KEYS, k_last));
      if constexpr (EB == 1) {
        ksc[0] *= a.c2;
        ksc[1] *= a.c2;
      }
      const float ks_next[2] = {ksn[0], ksn[1]};
      const bool edge = kb + PC_KEYS > min(w_lim + 1, k_hi) || ok != 15;
      pc_f32x16 sc[2] = {zero, zero};
      u32x4 ring[PC_AHEAD];
      float wt[16];                                             // a tile's weights
      u32x4 p[2], p_lo[2];                                      // and as two bf16 terms, 8 t .. + 7 of them
      auto split = [&](int t, int e) __attribute__((always_inline)) {
        const float w0 = wt[8 * t + 2 * e], w1 = wt[8 * t + 2 * e + 1];
        p[t][e] = pa_pack(w0, w1);
        p_lo[t][e] = pa_pack(w0 - bf16_lo(p[t][e]), w1 - bf16_hi(p[t][e]));
      };
      // the scores of key tile kt, scaled and masked; m moved if they pass it (what has it as its reference follows)
      auto finish = [&](int kt) __attribute__((always_inline)) {
        if constexpr (EB == 1) scale16(sc[kt], ksc[kt]);
        if (__builtin_expect(edge, 0)) {
          const int lim = min(rlim, k_hi - 1) - kb - 4 * hf;
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (32 * kt + 8 * (x >> 2) + (x & 3) > lim || !(ok >> (2 * kt + (x >> 3)) & 1)) sc[kt][x] = -INFINITY;
        }
        float top = sc[kt][0];
#pragma unroll
        for (int x = 1; x < 16; ++x) top = fmaxf(top, sc[kt][x]);
        if constexpr (EB == 2) top *= a.c2;
        if (__builtin_expect(__any(top - m > PA_SLACK), 0)) {
          const float x = fmaxf(top, __shfl_xor(top, 32, 64));  // of the row, in its two lanes
          const float mn = x - m > PA_SLACK ? x : m;
          const float f = __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= f;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n] *= f;
            __builtin_amdgcn_sched_barrier(0);                  // a tile of O at a time
          }
          if (kt == 1) {
#pragma unroll
            for (int x = 0; x < 16; ++x) wt[x] *= f;
#pragma unroll
            for (int e = 0; e < 4; ++e) split(0, e);
          }
        }
      };
      // weight x of tile kt, times its value's scale
      auto weight = [&](int kt, int x) __attribute__((always_inline)) {
        float w = __builtin_amdgcn_exp2f(EB == 2 ? fmaf(sc[kt][x], a.c2, -m) : sc[kt][x] - m);
        l += w;
        if constexpr (EB == 1) w *= row_lane_of(vsc[kt], x);
        asm volatile("" : "+v"(w));                             // evaluated here, beside a product
        wt[x] = w;
      };
#pragma unroll
      for (int x = 0; x < PC_AHEAD; ++x) ring[x] = operand(x);
#pragma unroll
      for (int st = 0; st < KS; ++st) {                         // beside the next step's K on its way to LDS
        sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_pa8(ring[st % PC_AHEAD]), as_pa8(qa[st]), sc[0], 0, 0, 0);
        ring[st % PC_AHEAD] = operand(st + PC_AHEAD);
#pragma unroll
        for (int z = st * KP / KS; z < (st + 1) * KP / KS; ++z) stage_k(to, z);
        __builtin_amdgcn_sched_barrier(0);
      }
      fetch_k();
      finish(0);
#pragma unroll
      for (int st = 0; st < KS; ++st) {                         // beside the other tile's weights
        const int x = KS + st;
        sc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_pa8(ring[x % PC_AHEAD]), as_pa8(qa[st]), sc[1], 0, 0, 0);
        ring[x % PC_AHEAD] = operand(x + PC_AHEAD);
#pragma unroll
        for (int y = st * 16 / KS; y < (st + 1) * 16 / KS; ++y) weight(0, y);
#pragma unroll
        for (int e = 0; e < 4; ++e)                             // halfway: the first eight are there
          if (st == KS / 2 + e * (KS / 8)) split(0, e);
        __builtin_amdgcn_sched_barrier(0);
      }
      finish(1);
      if (V_FIRST == 0) clean(kb + PC_KEYS, ok_next);
      // products y of V, two to an operand, beside the other tile's weights and the next step's V
      auto add_v = [&](int y) __attribute__((always_inline)) {
        const int x = 2 * KS + y, t = y / NT % 2;
        const u32x4 v = ring[x % PC_AHEAD];
        o[y % NT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_pa8(v), as_pa8(p[t]), o[y % NT], 0, 0, 0);
        o[y % NT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_pa8(v), as_pa8(p_lo[t]), o[y % NT], 0, 0, 0);
        if (x + PC_AHEAD < 2 * KS + 4 * NT) ring[x % PC_AHEAD] = operand(x + PC_AHEAD);
#pragma unroll
        for (int e = 0; e < 4; ++e)                             // the eight weights of the next NT products
          if (y < 3 * NT && y % NT == e * (NT / 4)) split(1 - t, e);
        if (y < 2 * NT)
#pragma unroll
          for (int z = y * 8 / NT; z < (y + 1) * 8 / NT; ++z) weight(1, z);
        if (y >= V_FIRST)
#pragma unroll
          for (int z = (y - V_FIRST) * VP / (4 * NT - V_FIRST); z < (y - V_FIRST + 1) * VP / (4 * NT - V_FIRST); ++z) stage_v(to, z);
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int y = 0; y < 2 * NT; ++y) add_v(y);
      if (V_FIRST != 0) clean(kb + PC_KEYS, ok_next);
#pragma unroll
      for (int y = 2 * NT; y < 4 * NT; ++y) add_v(y);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        ksc[kt] = ks_next[kt];
        vsc[kt] = vsn[kt];
      }
      fetch_v();
#pragma unroll
      for (int x = 0; x < KS && x < 8; ++x) k_at[x] ^= STAGE;
#pragma unroll
      for (int x = 0; x < 8; ++x) v_at[x >> 2][x & 3] ^= STAGE;
      ok = ok_next;
      ok_next = ok_further;
      __syncthreads();
    }

    // O through LDS, so that a row is written as consecutive bytes: 16-byte unit c of row r at c ^ (r % 16)
    l += __shfl_xor(l, 32, 64);
    const uint64_t none = __ballot(l == 0.0f);
    if (lane == 0) blank[wave] = (uint32_t)none;
    float* ob = reinterpret_cast<float*>(lds);
    const float inv = a.nsplit > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int y = 0; y < 16; y += 4) {
        const int c = 8 * n + (y >> 1) + hf;
        *reinterpret_cast<float4*>(ob + (32 * wave + li) * D + 4 * (c ^ (li & 15))) =
            make_float4(o[n][y] * inv, o[n][y + 1] * inv, o[n][y + 2] * inv, o[n][y + 3] * inv);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (a.nsplit > 1 && used && hf == 0)
      pa_ml(a, D)[((size_t)(s.first + i) * a.Hq + kh * GQ + g) * a.nsplit + split] = make_float2(m, l);
    __syncthreads();
    if (odd) {
      // a dim of a key that clean() set to 0 is NaN for the rows that see the key
      for (int key = max(k_lo, first_lim + 1); key < k_hi; ++key) {
        const int pg = pa_page(table, key >> a.c.shift);
        if (pg < 0 || pg >= a.c.n_pages) continue;
        const uint32_t at = (((uint32_t)pg * a.c.Hkv + kh) << a.c.shift) + (key & mask);
        bool bad = false;
        if constexpr (EB == 1) bad = !(fabsf(a.c.vs[at]) < INFINITY);
        if ((int)threadIdx.x < D) {
          const uint8_t* pv = a.c.v + (uint64_t)at * ROW + EB * threadIdx.x;
          if constexpr (EB == 2) bad = (*reinterpret_cast<const uint16_t*>(pv) & 0x7f80u) == 0x7f80u;
          if constexpr (FMT == QVEX_KV_FP8) bad |= (*pv & 0x7fu) == 0x7fu;
          if (bad)
            for (int rr = max((key - s.pos) * GQ, r0) - r0; rr <= last - r0; ++rr)
              ob[rr * D + 4 * ((threadIdx.x >> 2) ^ (rr & 15)) + (threadIdx.x & 3)] = __uint_as_float(0x7fc00000u);
        }
      }
      __syncthreads();
    }
#pragma unroll 1
    for (int x = threadIdx.x; x < (last + 1 - r0) * (D / 4); x += 256) {
      const int rr = x / (D / 4), c = x % (D / 4), tok = s.first + (r0 + rr) / GQ, head = kh * GQ + (r0 + rr) % GQ;
      const float4 v = *reinterpret_cast<const float4*>(ob + rr * D + 4 * (c ^ (rr & 15)));
      if (a.nsplit > 1) {
        *reinterpret_cast<float4*>(a.ws + (((size_t)tok * a.Hq + head) * a.nsplit + split) * D + 4 * c) = v;
      } else {
        const float y[4] = {v.x, v.y, v.z, v.w};
        PaGate(a, tok, head, 4 * c).store(a, tok, head, 4 * c, D, y, !(blank[rr >> 5] >> (rr & 31) & 1));
      }
    }
    __syncthreads();
  }

  // rows without a visible key in a call of one split: nobody else writes them
  if (a.nsplit == 1 && s.pos < 0) {
    for (int w = blk.tile; w < s.n && s.pos + w < 0; w += blk.tiles)
      for (int x = threadIdx.x; x < GQ * D; x += 256) a.out[((size_t)(s.first + w) * a.Hq + kh * GQ) * D + x] = 0;
  }
}

template <int FMT>
void launch(int D, dim3 grid, hipStream_t st, const PaArgs& a) {
  if (D == 256) hipLaunchKernelGGL((paged_chunk_kernel<FMT, 256>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((paged_chunk_kernel<FMT, 128>), grid, dim3(256), 0, st, a);
}

}  // namespace

void qvex::paged_chunk_attention(const void* args, int format, int D, int tiles, int B, void* stream) {
  const PaArgs& a = *static_cast<const PaArgs*>(args);
  const dim3 grid = pa_grid(a, B, tiles);
  const auto go = format == QVEX_KV_BF16 ? &launch<QVEX_KV_BF16> : format == QVEX_KV_INT8 ? &launch<QVEX_KV_INT8> : &launch<QVEX_KV_FP8>;
  go(D, grid, (hipStream_t)stream, a);
}
