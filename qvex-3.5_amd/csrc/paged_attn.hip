// Attention over a paged KV cache (mx.fast.scaled_dot_product_attention with the
// sigmoid gate, engine/model.py:221-232), pages in bf16 or 8 bits.
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q.k_p - m),  over positions p <= pos + i
//
// in one pass with a running reference m and sum, split over the keys and merged.
// A tile is 16 rows of one kv head: rows (position i, query head of the group),
// in that order, so that any group size fills it. Both products are transposed:
//   S^T[keys x rows] = K Q^T: row i of key tile h is key 8 (i / 4) + 4 h + i % 4 of a
//     32-key block, so that lane (lg, li) ends with keys 8 lg .. 8 lg + 7 of q row li, the B
//     operand of
//   O^T[dims x rows] += V^T P^T: lane (lg, li) of tile n holds keys 8 lg .. + 7 of dim
//     (D / 16) li + n. Those come from row-major pages without a transpose in memory: a
//     lane loads D / 16 consecutive dims of eight keys (16 lanes a whole row) and
//     gathers a dim's eight keys from its own registers.
// So K, V and P never leave their lanes, and a lane owns one q row. Codes are exact in
// bf16: K's scale multiplies the score, V's the weight. P goes into the second product
// as two bf16 terms (16 bits of it), so the output's own rounding is the one that shows.
//
// 16 query and 4 kv heads of 256, int8: 64 sequences of one row at up to 8192 keys read 618 MB in 130 to 136 us
// with a block per sequence and head (the CUs of the longest end last), in 117 and 6 of merging in equal runs (5.0
// TB/s; a plain read reaches 6.2). One row at 4096 keys 6.8 us and 3.3 to 4.4 of merging, four at 7001 (fp8) 11 and
// 3.5: two round trips of memory and two launches, on 132 and 112 blocks of 256 CUs and 16 and 64 of the merge.
#include "paged_attn.h"

namespace {

// One block per (kv head, 16-row tile, sequence, split): its 4 waves take 32 keys each of every
// 128, alone until their (m, l, O) are merged in LDS. PIPE (splits of several steps): the next
// step's K is asked for once the scores have this one's, its V behind the second product (us, 8
// sequences of up to 8192 keys in int8, one split each: 124 -> 95); a split of one step has no next.
// SHARES: one block per (kv head, run of the call's steps), which takes the parts of its run one after another.
template <int FMT, int D, bool PIPE, bool SHARES>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PaArgs a) {
#pragma clang fp contract(off)
  constexpr int EB = kv_bytes(FMT), KS = D / 32, KU = D * EB / 64, E = D / 16, VW = E * EB / 4, ROW = D * EB;
  __shared__ __align__(16) float obuf[4][PA_ROWS][D + 4];
  __shared__ float2 mlbuf[4][PA_ROWS];
  __shared__ int odd;                            // some V has a NaN or an infinity that not all rows see
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int li = lane & 15, lg = lane >> 4;
  const int GQ = a.Hq / a.c.Hkv, cap = a.r.width << a.c.shift, mask = (1 << a.c.shift) - 1, split = blockIdx.z;
  int b, kh, tile, tiles, k_lo, k_hi = 0;
  int at = 0, end = 0, before = 0, steps = 0;                     // SHARES: steps of the run, of the sequence in it
  if constexpr (SHARES) {
    kh = blockIdx.x % a.c.Hkv;
    int total = 0;
    for (int c = 0; c < a.B; c += 64) total += pa_wave_sum(c + lane < a.B ? pa_steps(a, c + lane, GQ) : 0);
    const int run = (total + a.shares - 1) / a.shares;
    at = (blockIdx.x / a.c.Hkv) * run;
    end = min(at + run, total);
    if (at >= end) return;
    b = a.B;
    for (int c = 0; c < a.B; c += 64) {
      const int mine = c + lane < a.B ? pa_steps(a, c + lane, GQ) : 0;
      int upto = mine;
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const int x = __shfl_up(upto, m, 64);
        upto += lane >= m ? x : 0;
      }
      const uint64_t past = __ballot(before + upto > at);
      if (past) {
        const int l = __builtin_ctzll(past);
        b = c + l;
        steps = __builtin_amdgcn_readlane(mine, l);
        before += __builtin_amdgcn_readlane(upto, l) - steps;
        break;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (b == a.B) return;                                         // only if positions change under the call
    tile = 0;
    tiles = 1;
    k_lo = (at - before) * PA_STEP;
  } else {
    const PaBlock blk(a);
    b = blk.b;
    kh = blk.kh;
    tile = blk.tile;
    tiles = blk.tiles;
    k_lo = split * a.kps;
  }
  KvSeq s(a.r, b);
  int rows = s.n * GQ;
  const int32_t* table = a.r.table + b * a.r.stride;
  // the first keys' pages, asked for beside the position (-0.4 us of a small call)
  auto page_at = [&](int kb) __attribute__((always_inline)) {
    return pa_page(table, min(kb >> a.c.shift, a.r.width - 1));
  };
  int first0 = page_at(k_lo + 32 * wave), first1 = page_at(k_lo + 32 * wave + 16);

  while (SHARES || tile * PA_ROWS < rows) {
    const int row = tile * PA_ROWS + li, last = min(rows, (tile + 1) * PA_ROWS) - 1;
    const bool used = row < rows;
    const int i = used ? row / GQ : 0, g = used ? row - i * GQ : 0;
    const int i_lo = tile * PA_ROWS / GQ, i_hi = last / GQ;       // positions of the tile
    const int rlim = used ? min(s.pos + i, cap - 1) : -1;
    const int keys = min(s.pos + i_hi + 1, cap);                  // that any row sees
    if constexpr (SHARES) {
      k_hi = tile ? keys : min((min(end, before + steps) - before) * PA_STEP, keys);
    } else {
      k_hi = split == a.nsplit - 1 ? keys : min(k_lo + a.kps, keys);
      if (k_lo >= k_hi) {                                         // uniform; the merge does not read it
        tile += tiles;
        continue;
      }
    }

    if (FMT != QVEX_KV_INT8) {
      if (threadIdx.x == 0) odd = 0;
      __syncthreads();
    }
    u32x4 qa[KS];
    const uint16_t* qp = a.q + (s.first + i) * a.q_token + (kh * GQ + g) * a.q_head;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const int d = EB == 2 ? 32 * st + 8 * lg : 64 * (st >> 1) + 16 * lg + 8 * (st & 1);
      qa[st] = used ? pa_load8(qp + d, a.vec) : u32x4{0, 0, 0, 0};
    }

    u32x4 kr[2][KU];
    uint32_t vr[8][VW];
    float ksc = 0.0f, vsc = 0.0f;                                 // lane e of 16: of key 8 lg + e
    bool ok0 = true, ok1 = true;                                  // of the block's two 16-key halves
    long at0 = 0, at1 = 0;
    auto locate = [&](int kb, int p0, int p1) __attribute__((always_inline)) {
      ok0 = p0 >= 0 && p0 < a.c.n_pages;
      ok1 = p1 >= 0 && p1 < a.c.n_pages;
      at0 = (((long)(ok0 ? p0 : 0) * a.c.Hkv + kh) << a.c.shift) + (kb & mask);
      at1 = (((long)(ok1 ? p1 : 0) * a.c.Hkv + kh) << a.c.shift) + ((kb + 16) & mask);
    };
    auto load_k = [&]() __attribute__((always_inline)) {
      const long at = (li >> 3 ? at1 : at0) + 8 * ((li >> 2) & 1) + (li & 3);
      const uint8_t* p = a.c.k + at * ROW + 16 * lg;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < KU; ++u) kr[h][u] = load16(p + 4 * h * ROW + 64 * u);
      if constexpr (EB == 1) {
        ksc = a.c.ks[(lg >> 1 ? at1 : at0) + 8 * (lg & 1) + (li & 7)];
      }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
      const long at = (lg >> 1 ? at1 : at0) + 8 * (lg & 1);
      const uint8_t* p = a.c.v + at * ROW + li * (4 * VW);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (VW == 2) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(p + e * ROW);
          vr[e][0] = w[0];
          vr[e][1] = w[1];
        } else {
#pragma unroll
          for (int u = 0; u < VW / 4; ++u) {
            const u32x4 w = load16(p + e * ROW + 16 * u);
#pragma unroll
            for (int x = 0; x < 4; ++x) vr[e][4 * u + x] = w[x];
          }
        }
      }
      if constexpr (EB == 1) vsc = a.c.vs[at + (li & 7)];
    };

    const pa_f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = PA_NONE, l = 0.0f;
    pa_f32x4 o[E];
#pragma unroll
    for (int n = 0; n < E; ++n) o[n] = zero;

    int kb = k_lo + 32 * wave, p0 = first0, p1 = first1;
    if (PIPE && kb < k_hi) {
      locate(kb, p0, p1);
      p0 = page_at(kb + PA_STEP);
      p1 = page_at(kb + PA_STEP + 16);
      load_k();
      load_v();
    }
    if (PIPE) {
#pragma unroll
      for (int st = 0; st < KS; ++st) asm volatile("" : "+v"(qa[st]));   // Q waited for here, not in the loop with all of V
    }
    for (; kb < k_hi; kb += PA_STEP) {
      if (!PIPE) {
        locate(kb, p0, p1);
        p0 = page_at(kb + PA_STEP);                               // the next step's
        p1 = page_at(kb + PA_STEP + 16);
        load_k();
        load_v();
      }
      const bool here0 = ok0, here1 = ok1;                        // of this step
      pa_f32x4 sc[2] = {zero, zero};
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 ka;
          if constexpr (EB == 2) ka = kr[h][st];
          else ka = codes8<FMT>(kr[h][st >> 1][2 * (st & 1)], kr[h][st >> 1][2 * (st & 1) + 1]);
          sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_pa8(ka), as_pa8(qa[st]), sc[h], 0, 0, 0);
        }
      if (PIPE) __builtin_amdgcn_sched_barrier(0);                // V is not touched (nor waited for) before its product
      float t[8], top = -INFINITY;
      uint32_t vis = 0xff;                                        // of the lane's keys 8 lg ..
      const bool edge = kb + 32 > min(s.pos + i_lo + 1, k_hi) || !here0 || !here1;   // uniform
      if (edge) {
        vis = 0;
        if (lg >> 1 ? here1 : here0)
#pragma unroll
          for (int e = 0; e < 8; ++e) vis |= (kb + 8 * lg + e <= min(rlim, k_hi - 1) ? 1u : 0u) << e;
      }
      const float kf = EB == 1 ? ksc * a.c2 : a.c2;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[e] = sc[e >> 2][e & 3] * (EB == 1 ? row_lane_of(kf, e) : kf);
        if (edge && !(vis >> e & 1)) t[e] = -INFINITY;
        top = fmaxf(top, t[e]);
      }
      if (PIPE) {
        // behind the last step of the wave this one again, so that the loads need no branch (a branch would have
        // their registers copied, and so waited for)
        const bool more = kb + PA_STEP < k_hi;
        const int kn = more ? kb + PA_STEP : kb;
        if (more) {
          locate(kn, p0, p1);
          p0 = page_at(kn + PA_STEP);
          p1 = page_at(kn + PA_STEP + 16);
        }
        load_k();
        __builtin_amdgcn_sched_barrier(0);
      }
      if (__any(top - m > PA_SLACK)) {
        float x = fmaxf(top, __shfl_xor(top, 16, 64));
        x = fmaxf(x, __shfl_xor(x, 32, 64));                      // of the row, in its four lanes
        const float mn = x - m > PA_SLACK ? x : m;
        const float f = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int n = 0; n < E; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][j] *= f;
      }
      u32x4 p, p_lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[e] = __builtin_amdgcn_exp2f(t[e] - m);
        l += t[e];
        if constexpr (EB == 1) {
          const float w = t[e] * row_lane_of(vsc, e);             // by all lanes: a lane that is off gives nothing
          t[e] = edge && !(vis >> e & 1) ? 0.0f : w;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = pa_pack(t[2 * e], t[2 * e + 1]);
        p_lo[e] = pa_pack(t[2 * e] - bf16_lo(p[e]), t[2 * e + 1] - bf16_hi(p[e]));
      }
      if (edge && FMT != QVEX_KV_INT8) {
        // what no row of the tile sees is not data, and 0 times a NaN or an infinity is none: keys past the last
        // row's (and pages that are not there) become 0. So does a NaN or an infinity that some rows do
        // not see: the rows that do are marked at the end
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = kb + 8 * lg + e;
          const bool live = key < k_hi && (lg >> 1 ? here1 : here0);
#pragma unroll
          for (int u = 0; u < VW; ++u) {
            const uint32_t w = live ? vr[e][u] : 0, w1 = key > s.pos + i_lo ? tame<FMT>(w) : w;
            any |= w1 != w;
            vr[e][u] = w1;
          }
        }
        if (any) odd = 1;
      }
#pragma unroll
      for (int n = 0; n < E; n += 2) {
        u32x4 a0, a1;
        gather2<FMT, VW>(vr, n / 2, a0, a1);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_pa8(a0), as_pa8(p), o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_pa8(a0), as_pa8(p_lo), o[n], 0, 0, 0);
        o[n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_pa8(a1), as_pa8(p), o[n + 1], 0, 0, 0);
        o[n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_pa8(a1), as_pa8(p_lo), o[n + 1], 0, 0, 0);
      }
      if (PIPE) load_v();
    }

    // the waves' sums, merged in the order of the waves
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (used) {
      if (lg == 0) mlbuf[wave][li] = make_float2(m, l);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < E; n += 4)                            // dims E (4 lg + j) + n of q row li
          *reinterpret_cast<float4*>(&obuf[wave][li][E * (4 * lg + j) + n]) =
              make_float4(o[n][j], o[n + 1][j], o[n + 2][j], o[n + 3][j]);
    }
    __syncthreads();
    const int here = last + 1 - tile * PA_ROWS;
    for (int x = threadIdx.x; x < here * (D / 4); x += 256) {
      const int rr = x / (D / 4), d = 4 * (x % (D / 4)), rw = tile * PA_ROWS + rr;
      const int tok = s.first + rw / GQ, head = kh * GQ + rw % GQ;
      float mm = PA_NONE;
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, mlbuf[w][rr].x);
      float ll = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 ml = mlbuf[w][rr];
        const float f = __builtin_amdgcn_exp2f(ml.x - mm);
        const float4 ov = *reinterpret_cast<const float4*>(&obuf[w][rr][d]);
        ll = fmaf(ml.y, f, ll);
        acc[0] = fmaf(ov.x, f, acc[0]);
        acc[1] = fmaf(ov.y, f, acc[1]);
        acc[2] = fmaf(ov.z, f, acc[2]);
        acc[3] = fmaf(ov.w, f, acc[3]);
      }
      if (FMT != QVEX_KV_INT8 && odd) {
        for (int key = max(k_lo, s.pos + i_lo + 1); key < k_hi && key <= s.pos + rw / GQ; ++key) {
          const int pg = table[key >> a.c.shift];
          if (pg < 0 || pg >= a.c.n_pages) continue;
          const uint8_t* pv = a.c.v + ((((long)pg * a.c.Hkv + kh) << a.c.shift) + (key & mask)) * ROW + d * EB;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            bool bad;
            if constexpr (EB == 2) bad = (reinterpret_cast<const uint16_t*>(pv)[e] & 0x7f80u) == 0x7f80u;
            else bad = (pv[e] & 0x7fu) == 0x7fu;
            if (bad) acc[e] = __uint_as_float(0x7fc00000u);
          }
        }
      }
      if (SHARES ? tile != 0 : a.nsplit == 1) {
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= inv;
        PaGate(a, tok, head, d).store(a, tok, head, d, D, acc, ll != 0.0f);
      } else {
        const size_t rec = SHARES ? ((size_t)kh * (a.shares + a.B) + blockIdx.x / a.c.Hkv + b) * PA_ROWS + rr
                                  : ((size_t)tok * a.Hq + head) * a.nsplit + split;
        *reinterpret_cast<float4*>(a.ws + rec * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) pa_ml(a, D)[rec] = make_float2(mm, ll);
      }
    }
    __syncthreads();
    if constexpr (SHARES) {
      if (at == before && (tile + 1) * PA_ROWS < rows) {          // more rows than L promised: all their keys, here
        ++tile;
        k_lo = 0;
      } else {
        at = min(end, before + steps);
        before += steps;
        steps = 0;
        while (at < end && steps == 0 && ++b < a.B) steps = pa_steps(a, b, GQ);
        if (steps == 0) break;
        s = KvSeq(a.r, b);
        rows = s.n * GQ;
        table = a.r.table + b * a.r.stride;
        tile = 0;
        k_lo = 0;
      }
      first0 = page_at(k_lo + 32 * wave);
      first1 = page_at(k_lo + 32 * wave + 16);
    } else {
      tile += tiles;
    }
  }

  // rows of sequences without a visible key (a negative position): nobody else writes them
  if (!SHARES && a.nsplit == 1 && s.pos < 0) {
    for (int w = PaBlock(a).tile; w < s.n && s.pos + w < 0; w += tiles)
      for (int x = threadIdx.x; x < GQ * D; x += 256) a.out[((size_t)(s.first + w) * a.Hq + kh * GQ) * D + x] = 0;
  }
}

// A call of more than 8 rows per sequence takes the chunk form (paged_chunk.hip) if a sequence's
// rows of a kv head fill half a block (a quarter on average, whatever L allows) and (query, key) pairs
// * D are worth its start and end, 8 us against 3. us, this form | that one, 16 query and 4 kv heads of 256 (pairs = T * Hq *
// max_keys), int8: 64 positions at 1000 keys (1.1M) 21 | 25, at 4000 (4.2M) 32 | 35, 512 at 0 (4.2M) 20 | 32,
// 8 x 64 at 1000 (8.7M) 37 | 42, 64 at 8000 (8.3M) 44 | 40, 8 x 64 at 4000 (33M) 97 | 72, 512 at 4000 (37M) 100 | 75; bf16: 64 at
// 4000 40 | 39, 8 x 64 at 1000 53 | 44, 512 at 4000 165 | 71; of 128, 4 and 2 heads, int8: 512 at 4000 (9.2M) 27 |
// 29, 12 x 100 at 1000 (5.3M) 24 | 25, 8 x 200 at 4000 (27M) 62 | 49. One bound for all formats, between theirs.
constexpr long PA_CHUNK_MIN = 64;
// Many sequences of one tile and of long contexts are cut into equal runs of steps, one per CU (two of 128 dims), in
// place of equal splits of each: a sequence far below max_keys leaves no CU idle, for a search in
// the positions and a second launch (4 us), and 2 us for each end of a sequence inside a run. us, splits | runs, lengths
// 1/8 .. 1 of max_keys | all of them max_keys, 16 and 4 heads of 256: int8 24 x 8192 55, 50 | 78, 80; 40 x 2 rows at
// 5000 60, 50 | 85, 85; 64 x 8192 131, 121 | 186, 194; bf16 64 x 8192 258, 223 | 360, 366; 16 x 8192 (64 tiles, int8)
// 35, 38 | 49, 53; 128 x 2000 (16 steps) 64, 71 | 99, 109; 8 heads of 128, int8: 32 x 8192 71, 56 | 95, 103.
constexpr int PA_SHARE_SEQS = 255;     // times 2^23 steps of a sequence: below 2^31
constexpr int PA_SHARE_STEPS = 24;     // of max_keys, at least
constexpr double PA_CHUNK_WORK = 5e6 * 256;

// A row's records merged; D / 4 lanes hold the row, four dims each, eight records requested
// at a time. WIDE: a block per row, whose groups of lanes take every 256 / (D / 4)-th record and
// are then merged in their order: few rows of many records are otherwise a chain of round trips
// (us, 16 rows of 33 records 10.4 -> 4.1, 64 of 28 -> 5.0; many rows of few records need the lanes).
template <int D, bool WIDE, bool SHARES>
__global__ __launch_bounds__(256) void paged_attn_merge_kernel(PaArgs a) {
#pragma clang fp contract(off)
  constexpr int LANES = D / 4, PER = 256 / LANES, BATCH = 8, STEP = WIDE ? PER : 1;
  __shared__ __align__(16) float part[WIDE ? PER : 1][D];
  __shared__ float2 pml[WIDE ? PER : 1];
  const int b = blockIdx.y, sub = threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES);
  const KvSeq s(a.r, b);
  const int cap = a.r.width << a.c.shift;
  const long rows = (long)s.n * a.Hq;
  // SHARES: the runs that have steps of the sequence, run0 .. run0 + runs - 1
  const int GQ = a.Hq / a.c.Hkv;
  int run0 = 0, runs = 0;
  if constexpr (SHARES) {
    const int lane = threadIdx.x & 63;
    int total = 0, before = 0, mine = 0;
    for (int c = 0; c < a.B; c += 64) {
      const int x = c + lane < a.B ? pa_steps(a, c + lane, GQ) : 0;
      total += x;
      before += c + lane < b ? x : 0;
      mine += c + lane == b ? x : 0;
    }
    total = pa_wave_sum(total);
    before = pa_wave_sum(before);
    mine = pa_wave_sum(mine);
    const int run = (total + a.shares - 1) / a.shares;
    if (mine) {
      run0 = before / run;
      runs = (before + mine - 1) / run + 1 - run0;
    }
  }
  const int each = WIDE ? 1 : PER;
  for (long w = (long)blockIdx.x * each + (WIDE ? 0 : sub); w < rows; w += (long)gridDim.x * each) {
    const int i = (int)(w / a.Hq), h = (int)(w - (long)i * a.Hq), tok = s.first + i;
    if (SHARES && i * GQ + h % GQ >= PA_ROWS) continue;           // its tile's block has written it
    const size_t rec = SHARES ? ((size_t)(h / GQ) * (a.shares + a.B) + run0 + b) * PA_ROWS + (i * GQ + h % GQ)
                              : ((size_t)tok * a.Hq + h) * a.nsplit;
    constexpr int GAP = SHARES ? PA_ROWS : 1;                     // from a row's record to its next
    const float2* mls = pa_ml(a, D) + rec;
    const float* os = a.ws + rec * D + d;
    float m = PA_NONE, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    // the first records are asked for before the position says how many there are (what the others hold is dropped)
    float2 ml[BATCH];
    float4 ov[BATCH];
    auto ask = [&](int s0, int n) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        const int at = min(s0 + x * STEP, n - 1);
        ml[x] = mls[at * GAP];
        ov[x] = *reinterpret_cast<const float4*>(os + (size_t)at * (GAP * D));
      }
    };
    if (!SHARES) ask(WIDE ? sub : 0, a.nsplit);
    const PaGate gate(a, tok, h, d);
    const int keys = min(s.pos + i + 1, cap);
    const int act = SHARES ? runs : keys <= 0 ? 0 : min((keys - 1) / a.kps + 1, a.nsplit);
    for (int s0 = WIDE ? sub : 0; s0 < act; s0 += BATCH * STEP) {
      if (SHARES || s0 >= BATCH * STEP) ask(s0, act);
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        if (s0 + x * STEP >= act) break;
        const float mn = fmaxf(m, ml[x].x);
        const float fa = __builtin_amdgcn_exp2f(m - mn), fb = __builtin_amdgcn_exp2f(ml[x].x - mn);
        m = mn;
        l = fmaf(ml[x].y, fb, l * fa);
        o[0] = fmaf(ov[x].x, fb, o[0] * fa);
        o[1] = fmaf(ov[x].y, fb, o[1] * fa);
        o[2] = fmaf(ov[x].z, fb, o[2] * fa);
        o[3] = fmaf(ov[x].w, fb, o[3] * fa);
      }
    }
    if constexpr (WIDE) {
      *reinterpret_cast<float4*>(&part[sub][d]) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) pml[sub] = make_float2(m, l);
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int x = 1; x < PER; ++x) m = fmaxf(m, pml[x].x);
        l = 0.0f;
        o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          const float f = __builtin_amdgcn_exp2f(pml[x].x - m);
          const float4 ov = *reinterpret_cast<const float4*>(&part[x][d]);
          l = fmaf(pml[x].y, f, l);
          o[0] = fmaf(ov.x, f, o[0]);
          o[1] = fmaf(ov.y, f, o[1]);
          o[2] = fmaf(ov.z, f, o[2]);
          o[3] = fmaf(ov.w, f, o[3]);
        }
      }
    }
    if (!WIDE || sub == 0) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= inv;
      gate.store(a, tok, h, d, D, o, l != 0.0f);
    }
    if constexpr (WIDE) __syncthreads();
  }
}

struct PaPlan {
  bool chunk;                          // paged_chunk.hip's form
  int tiles, kps, nsplit;              // row tiles of the longest sequence; keys per split; splits
  int shares;                          // or, in place of splits, runs of steps of all sequences
  uint64_t records;
  uint64_t bytes;
};

struct PaTiles {
  long tiles, blocks;                  // row tiles of the longest sequence, blocks with rows
};
PaTiles pa_tiles(bool chunk, int B, int L, int T, long GQ, int Hkv) {
  const int per = chunk ? qvex::PA_CHUNK_ROWS : PA_ROWS;
  const long most = std::min(L, std::max(T, 1)) * GQ, full = (long)T * GQ / per + B;   // tiles with rows, at most
  // where L says little of a sequence (every row of the call may be one's), few of B * tiles have rows: the blocks
  // of the longest sequence then take several
  const long tiles = std::min((most + per - 1) / per, std::max(4 * full, 4096L) / B + 1);
  return {tiles, std::max(std::min(B * tiles, full) * Hkv, 1L)};
}

// As many splits as give each CU a block (us, int8, 256-dim heads, blocks of one split | n splits: 16
// x 2000 keys (64 blocks) 28 | 4: 18 | 16: 22; 8 x 4 rows at 4096 (32) 54 | 8: 21 | 33: 30; 64 x 4600 (256) 112
// | 2: 112 | 36: 154). Never fewer for more steps.
long pa_splits(bool chunk, int L, long blocks, long steps) {
  const long want = chunk || L <= 8 ? 256 : 768;                  // many row tiles of unequal lengths
  long n = std::min(std::max(want / blocks, 1L), steps);
  if (!chunk && L <= 8) {
    // more of them, of 8 steps at least, where these leave a tenth of the CUs' rounds empty (us, as many as
    // fit once, so, sequences of unequal | of equal lengths: 24 x 8 rows at 8192 keys int8 104, 90 | 117, 133, bf16
    // 203, 162 | 230, 241; 40 x 8 at 3000 int8 71, 70 | 97, 91, bf16 139, 117 | 179, 159)
    double best = 0.0;
    for (long x = n, end = std::max(n, steps / 8); x <= end; ++x) {
      const double busy = (double)(x * blocks) / ((x * blocks + want - 1) / want * want);
      if (busy > best + 1e-9) {
        best = busy;
        n = x;
      }
      if (busy >= 0.9) break;
    }
  }
  return n;
}

bool pa_plan(int B, int L, int T, int Hq, int Hkv, int D, int max_keys, int kps, PaPlan* p) {
  if (B < 1 || L < 1 || T < 0 || Hkv < 1 || Hq < Hkv || Hq % Hkv || (D != 128 && D != 256) || max_keys < 1 ||
      max_keys > KV_LIMIT || kps < 0 || kps % PA_STEP)
    return false;
  const long GQ = Hq / Hkv, most = std::min(L, std::max(T, 1)) * GQ;
  p->chunk = L > 8 && most >= PA_CHUNK_MIN && (double)T * GQ >= 0.5 * PA_CHUNK_MIN * B &&
             (double)T * Hq * max_keys * D >= PA_CHUNK_WORK;
  const long steps = (max_keys + PA_STEP - 1) / PA_STEP;
  const PaTiles t = pa_tiles(p->chunk, B, L, T, GQ, Hkv);
  const bool chosen = kps == 0;
  if (chosen) {
    // two steps at least where a tile is more than half full (its records cost more than the second step: 4
    // rows at 7001 keys 16 | 14)
    const long least = !p->chunk && most > 8 && steps > 16 ? 2 : 1;
    const long n = pa_splits(p->chunk, L, t.blocks, steps);
    kps = (int)std::max((steps + n - 1) / n, least) * PA_STEP;
  }
  p->tiles = (int)std::min(t.tiles, 65535L);   // of a grid
  p->kps = kps;
  p->nsplit = (max_keys - 1) / kps + 1;
  p->shares = 0;
  p->records = p->nsplit == 1 ? 0 : (uint64_t)T * Hq * p->nsplit;
  if (chosen && !p->chunk && most <= PA_ROWS && B >= 2 && B <= PA_SHARE_SEQS && (long)B * Hkv >= 96 && steps >= PA_SHARE_STEPS) {
    p->shares = (int)std::max((D == 128 ? 512 : 256) / Hkv, 1);
    p->records = (uint64_t)Hkv * (p->shares + B) * PA_ROWS;
    p->nsplit = 1;
  }
  p->bytes = p->records * (D + 2) * sizeof(float);
  return true;
}

// Bytes that calls of these arguments and of any keys up to max_keys take: splits of whole steps are rounded, so
// that fewer keys can have more of them (16 query and 4 kv heads of 256, a row: 32 at 8192 keys, 18 at 9000).
uint64_t pa_most_bytes(int B, int L, int T, int Hq, int Hkv, int D, int max_keys, int kps) {
  PaPlan p;
  if (!pa_plan(B, L, T, Hq, Hkv, D, max_keys, kps, &p)) return 0;
  uint64_t records = p.records;
  if (kps == 0 && T > 0) {
    const long steps = (max_keys + PA_STEP - 1) / PA_STEP;
    const auto more = [&](bool chunk, long most) {
      const long n = pa_splits(chunk, L, pa_tiles(chunk, B, L, T, Hq / Hkv, Hkv).blocks, std::min(steps, most));
      if (n > 1) records = std::max(records, (uint64_t)T * Hq * n);
    };
    if (p.shares) more(false, PA_SHARE_STEPS - 1);                // the other form's calls are shorter
    else more(false, p.chunk ? (long)(PA_CHUNK_WORK / ((double)T * Hq * D)) / PA_STEP + 2 : steps);
    if (p.chunk) more(true, steps);
  }
  return records * (D + 2) * sizeof(float);
}

template <int FMT, int D>
void launch_attn(dim3 grid, hipStream_t st, const PaArgs& a) {
  // 16 KB of K and of V per wave leave no registers over: bf16 of 256 dims spills 6 registers without the prefetch, fp8 3
  // with it, around the loop of steps (two of bf16's accesses are in it under SHARES)
  constexpr bool FITS = FMT != QVEX_KV_BF16 || D == 128;
  // many rows: other tiles' waves hide the loads, and fewer registers are worth more (us, two rows' tiles or more, with |
  // without: 12 x 200 rows at 1500 keys 27.9 | 26.8; 2 x 64 at 1000 25.0 | 23.6; 16 x 12 at 2000 39.4 | 38.3)
  if (a.shares) hipLaunchKernelGGL((paged_attn_kernel<FMT, D, FITS, true>), grid, dim3(256), 0, st, a);
  else if (FITS && a.kps > PA_STEP && a.r.L <= 8)
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, FITS, false>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((paged_attn_kernel<FMT, D, false, false>), grid, dim3(256), 0, st, a);
}

}  // namespace

extern "C" uint64_t qvex_paged_attention_workspace_bytes(int B, int L, int T, int Hq, int Hkv, int D, int max_keys,
                                                         int keys_per_split) {
  return pa_most_bytes(B, L, T, Hq, Hkv, D, max_keys, keys_per_split);
}

extern "C" int qvex_paged_attention(const qvex_kv_pages* pages, const qvex_kv_rows* rows, const uint16_t* q,
                                    long q_token, long q_head, int Hq, int max_keys, int keys_per_split,
                                    const uint16_t* gate, long gate_token, long gate_head, float scale, uint16_t* out,
                                    void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* fn = "qvex_paged_attention";
  PaArgs a;
  if (const int rc = kv_check(fn, pages, rows, &a.c, &a.r)) return rc;
  const int B = rows->B, D = pages->D;
  PaPlan p;
  QVEX_CHECK_ARG(pa_plan(B, a.r.L, a.r.T, Hq, a.c.Hkv, D, max_keys, keys_per_split, &p) && Hq <= 16384,
                 "%s: Hq=%d Hkv=%d max_keys=%d keys_per_split=%d (a multiple of 128, or 0)", fn, Hq, a.c.Hkv, max_keys,
                 keys_per_split);
  QVEX_CHECK_ARG(p.nsplit <= 65535 && (long)B * a.c.Hkv < 1 << 24, "%s: grid too large", fn);
  QVEX_CHECK_ARG(scale >= 0.0f && scale < INFINITY, "%s: scale=%g must be finite, not negative", fn, (double)scale);
  if (a.r.T == 0) return QVEX_OK;
  QVEX_CHECK_ARG(q && out && qvex_aligned(q, 2) && qvex_aligned(out, 16) && qvex_aligned(gate, 2),
                 "%s: null or misaligned q, gate or out (out 16-byte aligned)", fn);
  QVEX_CHECK_ARG(workspace_bytes >= p.bytes && (p.bytes == 0 || (workspace && qvex_aligned(workspace, 16))),
                 "%s: workspace %llu < %llu bytes, or not 16-byte aligned", fn, (unsigned long long)workspace_bytes,
                 (unsigned long long)p.bytes);
  a.q = q;
  a.q_token = q_token;
  a.q_head = q_head;
  a.gate = gate;
  a.g_token = gate_token;
  a.g_head = gate_head;
  a.out = out;
  a.ws = (float*)workspace;
  a.Hq = Hq;
  a.kps = p.kps;
  a.nsplit = p.nsplit;
  a.records = p.records;
  a.B = B;
  a.shares = p.shares;
  a.vec = (q_token % 8 | q_head % 8) == 0 && qvex_aligned(q, 16);
  a.c2 = fmaxf(scale * 1.44269504088896340736f, 1e-37f);       // a masked score stays -inf at a scale of 0 too
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid = p.shares ? dim3(a.c.Hkv * p.shares) : pa_grid(a, B, p.tiles);
  const int f = pages->format;
  const auto go = D == 256 ? (f == QVEX_KV_BF16   ? &launch_attn<QVEX_KV_BF16, 256>
                              : f == QVEX_KV_INT8 ? &launch_attn<QVEX_KV_INT8, 256>
                                                  : &launch_attn<QVEX_KV_FP8, 256>)
                           : (f == QVEX_KV_BF16   ? &launch_attn<QVEX_KV_BF16, 128>
                              : f == QVEX_KV_INT8 ? &launch_attn<QVEX_KV_INT8, 128>
                                                  : &launch_attn<QVEX_KV_FP8, 128>);
  if (p.chunk) qvex::paged_chunk_attention(&a, f, D, p.tiles, B, stream);
  else go(grid, st, a);
  QVEX_CHECK_LAUNCH(fn);
  if (p.nsplit > 1 || p.shares) {
    // wide by the rows of a sequence alone, so that calls of up to 8 give a row the same bits
    const bool wide = a.r.L <= 8 || p.shares;
    const int per = wide ? 1 : 256 / (D / 4);
    const long most = (8192 + B - 1) / B, want = ((long)a.r.L * Hq + per - 1) / per;
    const dim3 mgrid((unsigned)std::min(want, most), B);
    const auto merge = p.shares ? (D == 256 ? &paged_attn_merge_kernel<256, true, true> : &paged_attn_merge_kernel<128, true, true>)
                       : D == 256 ? (wide ? &paged_attn_merge_kernel<256, true, false> : &paged_attn_merge_kernel<256, false, false>)
                                  : (wide ? &paged_attn_merge_kernel<128, true, false> : &paged_attn_merge_kernel<128, false, false>);
    hipLaunchKernelGGL(merge, mgrid, dim3(256), 0, st, a);
    QVEX_CHECK_LAUNCH("qvex_paged_attention/merge");
  }
  return QVEX_OK;
}
