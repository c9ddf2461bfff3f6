// Attention of the prompt encoder's kind: sequences of different lengths in one launch, grouped
// query heads, causal or full, k and v as packed token rows or in the pages of a cache.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),  s_ij = scale q_i . k_j,  m_i = max_j s_ij
// over the keys j that query i sees (lim_i of them: a prefix of its sequence); no key: o_i = 0.
//
// The G query heads that share a kv head are rows of one block: row r of sequence b is token r / G,
// head hk G + r % G. K and V are then read once for G heads, a single token still fills G rows of a
// matrix instruction, and a causal diagonal is G times narrower in rows.
//
// attn_seq_kernel: one work-group = 4 waves = 64 rows of one (sequence, kv head), 32-key tiles,
// double-buffered in LDS by buffer_load ... lds (32 KiB, three or four work-groups a CU: short sequences are
// bound by the latency of a chain of loads, which other work-groups fill). Per wave and tile, 16 rows:
//   S^T = K Q^T (mfma 16x16x32, K rows by ds_read_b128 from an XOR-swizzled image, Q^T in registers)
//   a lane holds 8 keys of one row: online softmax in log2 units (running max and sum in fp32, the
//   rescale only when a max grows by more than 2^8), P rounded to bf16 for the second product, as the
//   matrix instruction takes it (at most 2^-8 of the mean |v| that the row sees)
//   O^T += V^T P^T (V^T by ds_read_b64_tr_b16; the S^T registers are the P^T operand)
// Rows past a tile's last key come from the buffer's range check as zeros. Measured (device, median): 64 windows
// of 16 .. 64 rows, 16 heads of 80, 9.3 us (2.7 TB/s); six causal prompts of 70 .. 420, 28 heads over 4, 15.0 us, whose
// longest block walks 14 tiles one behind the other; one of 300 10.0; 784 rows of 16 heads of 80, all of which see
// each other, 15.9; 16 prompts of 400 44 us, 64 175 (420 TFLOP/s). Tried and
// slower or equal: 64-key tiles, three stages with one barrier a tile, 32 rows a wave, two groups of waves a
// block that share its keys, the next tile's scores beside this one's softmax.
#include <cmath>
#include <type_traits>

#include "attn_seq.h"

namespace {

constexpr int kBM = 64;  // rows of a work-group

template <bool PAGED, int NK, int WGS>  // NK 32-wide steps of the head: head_dim <= 32 NK; work-groups of a CU
__global__ void __launch_bounds__(256, WGS) attn_seq_kernel(SeqArgs a) {
  constexpr int ND = 2 * NK;     // 16-wide blocks of the output
  constexpr int KT = 32, KB = KT / 16, NP = KT / 16;  // keys of a tile, their blocks, pieces of a wave
  constexpr int TILE = KT * kRowB;
  __shared__ __attribute__((aligned(16))) char smem_raw[4 * TILE];  // K0 V0 K1 V1
  char QIE_LDS* smem = (char QIE_LDS*)smem_raw;

  const int hk = blockIdx.x % a.Hk;
  Item it;
  if (!find_item<PAGED, kBM>(a, blockIdx.x / a.Hk, it)) return;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int g = lane >> 4, ql = lane & 15;
  const int rows = it.n * a.G;
  const int last = (min(rows, (it.blk + 1) * kBM) - 1) / a.G;
  const int off = it.kv - it.n;
  const int most = a.causal ? min(it.kv, max(off + last + 1, 0)) : it.kv;
  const int ntot = (most + kKB - 1) / kKB;  // in the 64-key units that chunks are counted in
  const int t0 = PAGED && a.ct ? it.ch * a.ct * 2 : 0;
  const int t1 = min((most + KT - 1) / KT, PAGED && a.ct ? t0 + 2 * a.ct : INT32_MAX);
  const bool whole = !PAGED || !a.ct || ntot <= a.ct;
  if (t0 > 0 && t0 >= t1) return;  // a causal block that ends before this chunk

  // ---- tiles by LDS-DMA: a piece is 4 rows; wave w takes pieces w, w + 4, ... of K and of V. The
  // source chunk carries the XOR swizzle: K by the row, V by the row's low three bits, doubled
  const uint32_t ldb = (uint32_t)(a.ldk * 2);
  uint32_t ko[NP], vo[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int row = (wave + 4 * p) * 4 + g, ck = ql ^ (row & 15), cv = ql ^ ((row & 7) << 1);
    const uint32_t ro = (PAGED ? row & 15 : row) * ldb;  // pages: within the 16-row half that piece p lies in
    ko[p] = ck * 8 < a.Dh ? ro + ck * 16 : 0x80000000u;
    vo[p] = cv * 8 < a.Dh ? ro + cv * 16 : 0x80000000u;
  }
  const int64_t at0 = (int64_t)hk * a.hsk + (PAGED ? 0 : (int64_t)it.start * a.ldk);
  const int* table = PAGED ? a.table + (int64_t)it.b * a.ldt : nullptr;
  int tb = t0, pg[NP] = {};  // lane i: the pages of tile tb + i's halves (-1: outside the pool)
  auto pages = [&](int from) {
    tb = from;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int64_t page = ((int64_t)(from + lane) * KT + 16 * p) >> a.pshift;
      int id = -1;
      if (page < a.width) id = table[page];
      pg[p] = id >= 0 && id < a.pages ? id : -1;
    }
    __builtin_amdgcn_s_waitcnt(0);
  };
  auto dma = [&](int t, int st) {
    i32x4_t kr, vr;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if constexpr (PAGED) {
        const int key = t * KT + 16 * p, nrow = min(16, it.kv - key);
        const int id = __builtin_amdgcn_readlane(pg[p], t - tb);
        const bool ok = nrow > 0 && id >= 0;
        const int64_t at = at0 + (ok ? (int64_t)id * a.ps + (int64_t)(key & ((1 << a.pshift) - 1)) * a.ldk : 0);
        const int bytes = ok ? (nrow - 1) * (int)ldb + a.Dh * 2 : 0;
        kr = seq_rsrc(a.k + at, bytes);
        vr = seq_rsrc(a.v + at, bytes);
      } else if (p == 0) {
        const int64_t at = at0 + (int64_t)t * KT * a.ldk;
        const int bytes = (min(KT, it.kv - t * KT) - 1) * (int)ldb + a.Dh * 2;  // zeros past the sequence
        kr = seq_rsrc(a.k + at, bytes);
        vr = seq_rsrc(a.v + at, bytes);
      }
      const int r0 = (wave + 4 * p) * 4;
      seq_dma(kr, smem + (2 * st) * TILE + r0 * kRowB, ko[p]);
      seq_dma(vr, smem + (2 * st + 1) * TILE + r0 * kRowB, vo[p]);
    }
  };
  if (t0 < t1) {
    if constexpr (PAGED) pages(t0);
    dma(t0, 0);
    if (t0 + 1 < t1) dma(t0 + 1, 1);
  }

  const int r = it.blk * kBM + wave * 16 + ql;
  const int tok = min(r, rows - 1) / a.G, head = hk * a.G + min(r, rows - 1) % a.G;
  const int lim = a.causal ? min(it.kv, max(off + tok + 1, 0)) : it.kv;  // keys that this row sees
  const int lim0 = uni(lim);                                             // fewest of the wave
  bf16x8_t qf[NK];
  const bf16_t* qr = a.q + (int64_t)(it.start + tok) * a.ldq + (int64_t)head * a.hsq;
#pragma unroll
  for (int ks = 0; ks < NK; ++ks) {
    qf[ks] = bf16x8_t{};
    if (32 * ks + 8 * g < a.Dh) qf[ks] = *(const bf16x8_t*)(qr + 32 * ks + 8 * g);
  }
  f32x4_t o[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db) o[db] = f32x4_t{};
  float m_run = a.low, l_run = 0.f;
  float above = kRescale, mscale = a.c;  // seq_far

  __builtin_amdgcn_s_waitcnt(0);  // q and two tiles: from here on the counter is the tiles'
  asm volatile("s_barrier" ::: "memory");
  // one tile; MASKED: some row of the wave does not see all of it
  auto tile = [&](auto masked_t, int t) {
    constexpr bool MASKED = decltype(masked_t)::value;
    const char QIE_LDS* kt = smem + (2 * (t & 1)) * TILE;  // t0 is even
    const char QIE_LDS* vt = kt + TILE;
    f32x4_t s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      s[kb] = f32x4_t{};
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        const bf16x8_t A = *(const bf16x8_t QIE_LDS*)(kt + (kb * 16 + ql) * kRowB + (((4 * ks + g) ^ ql) << 4));
        s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, qf[ks], s[kb], 0, 0, 0);
      }
    }
    // V^T fragment: lane's d = 16 db + ql, keys 4 g + 0..3 and 16 further
    auto vfrag = [&](int db) -> bf16x8_t {
      const int row = 4 * g + (ql >> 2);
      const int ch = (2 * db + ((ql & 3) >> 1)) ^ ((row & 7) << 1);
      const char QIE_LDS* p0 = vt + row * kRowB + (ch << 4) + 8 * (ql & 1);
      const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t QIE_LDS*)p0);
      const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t QIE_LDS*)(p0 + 16 * kRowB));
      return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // V is read ahead of the exponentials; where four work-groups of 128-wide heads share a CU, a masked tile has
    // no registers to keep it in (184 bytes spilled, 318 us in place of 174 for 64 prompts of 400)
    constexpr bool KEEP = !MASKED || NK < 4 || WGS < 4;
    bf16x8_t vv[ND];
    if constexpr (KEEP) {
#pragma unroll
      for (int db = 0; db < ND; ++db) vv[db] = vfrag(db);
      asm volatile("" ::: "memory");
    }
    auto v_of = [&](int db) -> bf16x8_t {
      if constexpr (KEEP) return vv[db];
      else return vfrag(db);
    };
    const int kv0 = t * KT;
    if constexpr (MASKED) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kv0 + kb * 16 + 4 * g + i >= lim) s[kb][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = quad_max(mx);
    if (__any((mx - m_run) * a.c > above)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * a.c);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < ND; ++db) o[db] *= alpha;
      if (__builtin_expect(seq_far(a, m_run, above, mscale), 0))
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] -= m_run;
    }
    const float mc = m_run * mscale;
    bf16x8_t pf;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][i & 3], a.c, -mc));
      pf[i] = (__bf16)p[i];
    }
    l_run += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    asm volatile("" : "+v"(l_run));  // here, not behind the products
    // 0 * inf and 0 * NaN: a masked key's V must not reach the rows that do not see it
    bool bad = false;
    if constexpr (MASKED) {
      Magnitude mag;
#pragma unroll
      for (int db = 0; db < ND; ++db) mag.add(v_of(db));
      if constexpr (!KEEP) asm volatile("" ::: "memory");
      bad = __any(mag.nonfinite());
    }
    if (__builtin_expect(bad, 0)) {
      // the finite values as ever, then what a row sees of the others
#pragma unroll
      for (int db = 0; db < ND; ++db) {
        if constexpr (!KEEP) asm volatile("" ::: "memory");
        o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(finite(v_of(db)), pf, o[db], 0, 0, 0);
      }
#pragma unroll 1
      for (int j = 0; j < KT; ++j) {
        const char QIE_LDS* vr = vt + j * kRowB + 8 * (g & 1);
        const bool see = kv0 + j < lim;
#pragma unroll
        for (int db = 0; db < ND; ++db) {
          const u32x2_t w = *(const u32x2_t QIE_LDS*)(vr + (((2 * db + (g >> 1)) ^ ((j & 7) << 1)) << 4));
#pragma unroll
          for (int i = 0; i < 4; ++i) o[db][i] += special(i < 2 ? w.x : w.y, i & 1, see);
        }
      }
    } else {
#pragma unroll
      for (int db = 0; db < ND; ++db) o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v_of(db), pf, o[db], 0, 0, 0);
    }
    if (t + 1 == t1) return;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // this tile's stage is free
    if (t + 2 < t1) {
      if constexpr (PAGED)
        if (t + 2 - tb >= 64) pages(t + 2);
      dma(t + 2, t & 1);
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * NP) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    }
  };
  // the tiles that all rows of the wave see, then the others: one loop with a branch moved O between registers
  // and cost a third more instructions a tile. The waves change over apart, their barriers are the same.
  int t = t0;
#pragma unroll 1
  for (const int seen = min(t1, lim0 / KT); t < seen; ++t) tile(std::false_type{}, t);
#pragma unroll 1
  for (; t < t1; ++t) tile(std::true_type{}, t);

  const float l = quad_sum(l_run);
  if (r >= rows) return;
  if (!whole) {
    const int64_t pi = ((int64_t)(it.start + tok) * a.H + head) * a.maxch + it.ch;
    float* po = a.ws + pi * a.Dh;
#pragma unroll
    for (int db = 0; db < ND; ++db)
      if (16 * db + 4 * g < a.Dh) *(f32x4_t*)(po + 16 * db + 4 * g) = o[db];
    if (g == 0) *(f32x2_t*)(a.ws + (int64_t)a.T * a.H * a.maxch * a.Dh + pi * 2) = f32x2_t{m_run, l};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  bf16_t* dst = a.out + (int64_t)(it.start + tok) * a.ldo + (int64_t)head * a.hso;
#pragma unroll
  for (int db = 0; db < ND; ++db)
    if (16 * db + 4 * g < a.Dh)
      *(u32x2_t*)(dst + 16 * db + 4 * g) = u32x2_t{pack2(o[db][0] * inv, o[db][1] * inv),
                                                   pack2(o[db][2] * inv, o[db][3] * inv)};
}

// Joins the chunks of a row: o = sum_c w_c o_c / sum_c w_c l_c, w_c = exp2((m_c - max m) c). One wave a
// (token, head); the rows that one chunk held are written already. Bound by the latency of its loads, one behind
// the other: the length, then a lane's (m, l) and the first eight chunks' parts together, then eight at a time
// ahead of their use.
__global__ void __launch_bounds__(256) attn_seq_join_kernel(SeqArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + uni(threadIdx.x >> 6);
  if (row >= (int64_t)a.T * a.H) return;
  const int token = (int)(row / a.H), head = (int)(row - (int64_t)token * a.H);
  // the sequence of this token: the last one that starts at or before it
  int b = -1, start = 0, n = 0, kv = 0;
  if (!a.cu) {
    b = token;
    seq_span<true>(a, b, start, n, kv);
  }
  for (int b0 = 0; a.cu && b0 < a.B; b0 += 64) {
    int s0 = 0, n0 = 0, k0 = 0;
    if (b0 + lane < a.B) seq_span<true>(a, b0 + lane, s0, n0, k0);
    const unsigned long long hit = __ballot(b0 + lane < a.B && s0 <= token && token < s0 + n0);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      b = b0 + l;
      start = __builtin_amdgcn_readlane(s0, l);
      n = __builtin_amdgcn_readlane(n0, l);
      kv = __builtin_amdgcn_readlane(k0, l);
      break;
    }
  }
  if (b < 0) return;  // behind the last sequence
  // the row's block saw the keys of its last token: chunks as attn_seq_kernel cut them
  const int r = (token - start) * a.G + head % a.G, blk = r / a.bm;
  const int last = (min(n * a.G, (blk + 1) * a.bm) - 1) / a.G;
  const int most = a.causal ? min(kv, max(kv - n + last + 1, 0)) : kv;
  const int ntot = (most + kKB - 1) / kKB, nch = uni((ntot + a.ct - 1) / a.ct);
  if (nch <= 1) return;
  const float* pml = a.ws + (int64_t)a.T * a.H * a.maxch * a.Dh + row * a.maxch * 2;
  const int d = 2 * lane;
  const float* po = a.ws + row * a.maxch * a.Dh + (d < a.Dh ? d : 0);
  constexpr int kAhead = 8;
  f32x2_t ml = f32x2_t{a.low, 0.f}, v[kAhead], w[kAhead];
  if (lane < nch) ml = *(const f32x2_t*)(pml + 2 * lane);
  auto fetch = [&](f32x2_t* to, int from) {  // past the last chunk: the last once more, its weight is 0 then
#pragma unroll
    for (int i = 0; i < kAhead; ++i) to[i] = *(const f32x2_t*)(po + (int64_t)min(from + i, nch - 1) * a.Dh);
  };
  fetch(v, 0);
  float mx = ml[0];
  for (int c = lane + 64; c < nch; c += 64) mx = fmaxf(mx, pml[2 * c]);
  mx = wave_max(mx);
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int c0 = 0; c0 < nch; c0 += 64) {  // a lane weighs a chunk, then all lanes add 64 chunks' rows
    if (c0 > 0) {
      ml = f32x2_t{a.low, 0.f};
      if (c0 + lane < nch) ml = *(const f32x2_t*)(pml + 2 * (c0 + lane));
    }
    const float wt = c0 + lane < nch ? __builtin_amdgcn_exp2f((ml[0] - mx) * a.c) : 0.f;
    l = __builtin_fmaf(wt, ml[1], l);
    const int n64 = min(64, nch - c0);
    for (int c = 0; c < n64; c += kAhead) {
      fetch(w, c0 + c + kAhead);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float wc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wt), c + i));
        if (c + i < n64) {
          o0 = __builtin_fmaf(wc, v[i][0], o0);
          o1 = __builtin_fmaf(wc, v[i][1], o1);
        }
        v[i] = w[i];
      }
    }
  }
  l = wave_sum(l);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if (d < a.Dh) *(uint32_t*)(a.out + (int64_t)token * a.ldo + (int64_t)head * a.hso + d) = pack2(o0 * inv, o1 * inv);
}

// Which kernel, and how the keys are cut, by what the host knows: tokens, sequences, heads and the
// longest cache that a table can hold (packed sequences: their mean length). Rows are those of one kv
// head, tokens * G; a group is a (row block, kv head). Times in us (device, median), bf16, head_dim 128, 28 heads
// over 4 unless said, the other side in brackets.
//   few rows (attn_seq_few), 16-row blocks: up to 256 groups with eight waves each (one prompt of 100 tokens 5.9
//     [6.9 in 64-row blocks, 5.5 with four]), up to 512 with four, two a CU (one prompt of 200: 7.1 [9.9 with eight, 8.1
//     in 64-row blocks]; of 280: 8.2 [9.3]; past it, one of 300: 10.0 in 64-row blocks [10.4]), and more than that over up
//     to 1500 keys (80 tokens of 24 heads over 24, caches of 20, 300 and 1000: 15, 47 and 171 [26, 59 and 172 with eight];
//     over 2000 and 8000: 333 and 1284 with eight [335 and 1291]). 32-row blocks over more than 256 keys where 16-row ones
//     would be more than 256 (200 new tokens over 1000: 14.0 [15.3 in 16-row, 26.0 in 64-row blocks]; 10 x 20 over 300, 16
//     heads of 80, 7.7 [8.9]; over 400 the 200 would take 9.2 in 16-row ones [10.6]), or where a cache is read again for each 16 rows and that takes longer than the second half of a block: for
//     17 .. 32 rows a sequence from groups * keys = 6e4 on (3 new tokens over 6000 keys of one sequence 10.8 in 16-row
//     blocks [12.5], over 20000 17.7 in 32-row ones [21.5]; 4 over 20000 of 16 sequences 138 [194]), for more rows from 4e5
//     (8 over 20000 of one sequence: 21.0 in 16-row blocks [22.8]), and up to 1.5e6 against larger blocks (70 over 20000:
//     68 [94 in 64-row ones]; 100: 79 in 256-row ones [128]).
//   64-row blocks (attn_seq): shorter packed sequences (16 prompts of 400: 43 [53 in 256-row blocks]; from 200 groups
//     on very short ones, 16 x 30, 16 heads of 80: 4.7 [5.9 in 16-row blocks]), a short
//     cache's many rows (16 x 100 new tokens over 300: 19.5 [22.5 in 256-row blocks]), and 33 .. 64 rows of a sequence
//     over a long one where 32-row ones are more than 3e5 groups * keys (3 x 8 new tokens over 20000: 31 [59]; 16 x 8 135
//     [203]).
//   256-row blocks (attn_seq_pp) for packed sequences where there are 200 of them (2 x 1150, 252: 37 [39 in 64-row
//     blocks]; 4 x 650, 182: 29 in 64-row ones [31]), their rounds of 256 are two thirds full (2 x 1600, 350: 49 [55]; 2 x
//     1371, 300: level at 48), and the mean length is at least
//       head_dim      causal, shared heads          causal, not shared             full
//       97 .. 128     1000 (10 x 1000 107 [109],    2300 (24, 4 x 2500 189 [204],  800 (32 over 8, 29 of 570 .. 1084
//                     8 x 1300 129 [135],           4 x 1800 152 [123])            466 [491]; 4 x 700 52 [45])
//                     8 x 900 80 [76])
//       65 .. 96      1800 (16 over 2, 8 x 1800     2300 (16, 4 x 2500 113 [117],  900 (16, 8 x 900 61 [64],
//                     113 [119], 8 x 1400 79 [78])  4 x 2000 91 [81])              8 x 800 54 [50])
//       .. 64         3500 (12 over 4, 8 x 3500     6500 (8, 4 x 7000 289 [297],   1500 or 2700 (12 over 4, 6 x 1500 69 [70],
//                     level at 235, 4 x 4500        5 x 6000 307 [281])            6 x 1200 57 [51]; 8, 5 x 3000 123 [146],
//                     175 [187])                                                   8 x 2500 156 [155])
//     (narrow heads cost them as much as wide ones, and where heads share nothing a causal block spans 256 tokens). Over a
//     cache, for more than 2048 keys (6 x 600 over 3000: 174 [185]; 3 x 1500 over 1500: 85 [75]; heads
//     of 64 4096), where little of a block is padding: a sixth (6 x 600 over 3000, 16 heads of 80, 18 blocks for 14:
//     157 [104]), a third where shares even out the rest (10 of up to 758 over up to 9770: 423 [548]; 6 x 600 over 5000,
//     16 heads of 80, 176 [172]; past it, 20 x 160 over 5000, 16 heads: 265 [239]).
constexpr double kMostParts = 256 << 20;
struct SeqPlan {
  int bm, waves, ct, maxch, shares;
};

SeqPlan seq_plan(int tokens, int seqs, int heads, int kv_heads, int head_dim, bool causal, int64_t table_keys) {
  const bool paged = table_keys > 0;
  const double rows = (double)tokens * (heads / kv_heads), per = rows / seqs;  // in all, of a sequence
  const double keys = paged ? (double)table_keys : (double)tokens / seqs;
  const double g16 = kv_heads * fmax(seqs, rows / 16), g32 = kv_heads * fmax(seqs, rows / 32),
               g64 = kv_heads * fmax(seqs, rows / kBM), g256 = kv_heads * fmax(1.0, rows / kPPRows);
  const double r16 = (double)kv_heads * seqs * ceil(per / 16), r32 = (double)kv_heads * seqs * ceil(per / 32);  // as rounded
  const int few16 = r16 <= 256 ? 8 : 4;
  // from what length on 256-row blocks pay, and how full their rounds of 256 are
  const bool shared = heads > kv_heads;
  const double longest = head_dim > 64 ? (!causal ? (head_dim > 96 ? 800 : 900) : !shared ? 2300 : head_dim > 96 ? 1000 : 1800)
                         : shared      ? (causal ? 3500 : 1500)
                                       : (causal ? 6500 : 2700);
  const double rounds = ceil(g256 / 256), pad = ceil(per / kPPRows) * kPPRows / per;
  SeqPlan p{kBM, few16, 0, 1, 0};
  if (!paged) {
    if (g16 <= 512 && !(keys <= 100 && g16 >= 200)) p.bm = 16;
    else if (keys >= longest && g256 >= 200 && (g256 >= 512 || g256 >= 0.65 * 256 * rounds)) p.bm = kPPRows;
    return p;
  }
  if (per <= 16) {
    p.bm = 16;
    p.waves = keys <= 1536 ? few16 : 8;
  } else if (keys <= 512) {
    p.bm = r16 <= 256 ? 16 : r32 <= 256 && keys > 256 ? 32 : g16 <= 512 ? 16 : kBM;
    if (p.bm == 32) p.waves = 8;
  } else if (per > 32 && per <= 64 && g32 * keys > 3e5) {
    p.bm = kBM;
  } else if (per <= 32 || (g32 <= 512 && g32 * keys <= 1.5e6)) {
    p.bm = r16 <= 256 && g16 * keys <= (per <= 32 ? 6e4 : 4e5) ? 16 : 32;
    if (p.bm == 32) p.waves = 8;
  } else {
    p.bm = keys > (head_dim > 64 ? 2048 : 4096) && pad <= (keys > 4096 ? 1.5 : 1.2) ? kPPRows : kBM;
  }
  // Cuts: groups that do not fill the chip share a row's keys, in chunks whose fp32 parts a second kernel
  // joins: as many as fit 256 CUs at once (1000 new tokens over 4000 keys, two chunks: 86 [uncut 111, three
  // chunks 106]; three 64-row work-groups fit a CU), of 8 tiles at least; two also where they are up to 290 (1250 over
  // 4000, 278: 108 [111 uncut]; 1400, 308: 111 uncut [119]). Up to 1024 keys, none (one token over
  // 800: 7.8 in one launch [8.7 in two]). Few rows: 0.6 sqrt(tiles) tiles and 4 at least, where a chunk's time and
  // the join's meet (one token over 2000, 8000 and 32768 keys: 9.0, 11.2 and 19.4 [10.4, 12.6 and 20.9 with 8 and
  // 1.4 sqrt(tiles)]). Long tables are cut all the same, so that a long sequence among short ones is shared (48
  // tokens over 900 .. 32768 keys: 167 [326 uncut]): into 32 tiles (4 new tokens over 20000 keys of 16 sequences: 138
  // [146 with 64]), 64 where there is one sequence or the groups fill the chip without a cut. The cuts go by the table:
  // 16 tokens over 70 .. 600 keys take 7.1 in a table of that width, 9.1 in one of 2560 .. 32768 keys, 18.6 in one of
  // 131072.
  const double tiles = (double)((table_keys + kKB - 1) / kKB);
  if (tiles <= 16 || (p.bm == kBM && tiles <= 32)) return p;
  const double half = per > 16 ? 0.5 * seqs * kv_heads : 0;  // sequences end inside a block
  const double groups = p.bm == 16 ? g16 + half : p.bm == 32 ? g32 + half : p.bm == kBM ? g64 / 3 : g256 + half;
  // Many rows over more than 4096 keys, half of them kept at least: equal shares of the call's work (1500, 1100 and
  // 700 new tokens over 24000, 11000 and 7000: 715 [814 in chunks of 64 tiles]; 8 x 300 over 3000 and 9000: 242 [270];
  // of one length, 8 x 200 over 5000, the kernel goes back to whole blocks: 147 [138 without the line]). One sequence
  // too, also where its blocks fill their rounds (383 of them, 3500 new tokens over 24000: 1030 [1205 whole]; 256 of
  // them, 2340 tokens: 710 [700 whole, 793 in chunks]). From 512 blocks on whole ones even out (4 x 2000 over 2000 ..
  // 9000: 515 [615 in shares]). The sum of all blocks' keys has to fit the shares' 32 bits.
  if (p.bm == kPPRows && tiles > 64 && keys * seqs >= 2.0 * tokens && (g256 + seqs) * (keys + tokens + 1024) < 3e10 &&
      groups < 512) {
    p.shares = kv_heads <= 256 ? 256 / kv_heads : 1;
    return p;
  }
  if (p.bm == kPPRows && groups >= 512) return p;
  double n = fmax(1.0, floor(256 / groups));
  if (n == 1 && 2 * groups <= 290) n = 2;
  const double low = p.bm < kBM ? fmax(4.0, 0.6 * sqrt(tiles)) : 8;
  double ct = fmax(tiles / n, low);
  if (per <= 64 || tiles > 128) ct = fmin(ct, groups >= 256 || (per > 64 && seqs == 1) ? 64 : fmax(32.0, low));
  // The parts go by what the table could hold, for the lengths are not known here: kMostParts bytes of them at most.
  // Where fewer than two chunks of them fit, q alone is 64 MiB: thousands of blocks, no cut needed to fill the chip.
  const double fit = floor(kMostParts / ((double)tokens * heads * (head_dim + 2) * 4));
  if (fit < 2) return p;
  ct = fmax(ct, tiles / fit);
  if (tiles > ct) {
    p.ct = (int)ceil(tiles / ceil(tiles / ct - 1e-9));  // chunks of one size
    p.maxch = (int)ceil(tiles / p.ct);
  }
  return p;
}

template <bool PAGED>
int launch(const SeqArgs& a, unsigned grid, hipStream_t s) {
  // 128-wide heads fit four work-groups a CU with a register spilled (where V holds infinities): taken where more
  // than three a CU are there (64 prompts of 400: 174 us [184 with three]; six of 70 .. 420 18.5 [18.2 with three])
  if (a.Dh <= 64) attn_seq_kernel<PAGED, 2, 4><<<grid, 256, 0, s>>>(a);
  else if (a.Dh <= 96) attn_seq_kernel<PAGED, 3, 4><<<grid, 256, 0, s>>>(a);
  else if (grid > 3 * 256) attn_seq_kernel<PAGED, 4, 4><<<grid, 256, 0, s>>>(a);
  else attn_seq_kernel<PAGED, 4, 3><<<grid, 256, 0, s>>>(a);
  return qie_last_error();
}

int launch_seq(SeqArgs& a, const SeqPlan& p, bool paged, hipStream_t s) {
  a.bm = p.bm;
  a.ct = p.ct;
  a.maxch = p.maxch;
  a.shares = p.shares;
  if (p.bm != kBM) {
    const int rc = p.bm == kPPRows ? qie_launch_seq_pp(a, paged, s) : qie_launch_seq_few(a, paged, p.waves, s);
    if (rc) return rc;
  } else {
    const int64_t rb = (int64_t)a.T * a.G / kBM + a.B;  // at least the row blocks of any lengths
    const int64_t grid = rb * a.maxch * a.Hk;
    if (grid > INT32_MAX) return QIE_ERR_UNSUPPORTED;
    const int rc = paged ? launch<true>(a, (unsigned)grid, s) : launch<false>(a, (unsigned)grid, s);
    if (rc) return rc;
  }
  if (p.ct) attn_seq_join_kernel<<<(unsigned)(((int64_t)a.T * a.H + 3) / 4), 256, 0, s>>>(a);
  return qie_last_error();
}

void set_scale(SeqArgs& a, float scale) {
  a.c = scale * 1.4426950408889634f;
  a.low = -3e38f / fmaxf(a.c, 1.f);
}

bool seq_common_ok(const void* q, int64_t ldq, int64_t hsq, const void* k, const void* v, int64_t ldk, int64_t hsk,
                   int seqs, int tokens, int heads, int kv_heads, int head_dim, float scale, const void* out,
                   int64_t ldo, int64_t hso) {
  if (!(q && k && v && out && seqs > 0 && tokens >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0)) return false;
  if (!(head_dim > 0 && head_dim <= 128 && head_dim % 8 == 0 && scale > 0.f && scale <= 65536.f)) return false;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16 != 0) return false;
  if ((ldq | hsq | ldk | hsk | ldo | hso) % 8 != 0) return false;
  if (ldq < 0 || hsq < 0 || ldk < head_dim || ldk > (1 << 23) || hsk < 0 || ldo < head_dim || hso < head_dim) return false;
  return (int64_t)tokens * heads <= INT32_MAX / 2;
}

}  // namespace

extern "C" int qie_attention_packed_bf16(const void* q, int64_t ldq, int64_t hsq, const void* k, const void* v,
                                         int64_t ldk, int64_t hsk, const int* cu_seqlens, int seqs, int tokens,
                                         int heads, int kv_heads, int head_dim, int causal, float scale, void* out,
                                         int64_t ldo, int64_t hso, qie_stream_t stream) {
  QIE_CHECK_ARG(seq_common_ok(q, ldq, hsq, k, v, ldk, hsk, seqs, tokens, heads, kv_heads, head_dim, scale, out, ldo, hso));
  QIE_CHECK_ARG(cu_seqlens);
  if (tokens == 0) return QIE_OK;
  SeqArgs a{};
  a.q = (const bf16_t*)q; a.ldq = ldq; a.hsq = hsq;
  a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.ldk = ldk; a.hsk = hsk;
  a.out = (bf16_t*)out; a.ldo = ldo; a.hso = hso;
  a.cu = cu_seqlens;
  a.B = seqs; a.T = tokens; a.H = heads; a.Hk = kv_heads; a.G = heads / kv_heads; a.Dh = head_dim;
  a.causal = causal != 0;
  set_scale(a, scale);
  return launch_seq(a, seq_plan(tokens, seqs, heads, kv_heads, head_dim, causal != 0, 0), false, (hipStream_t)stream);
}

extern "C" int qie_attention_paged_workspace(int tokens, int seqs, int heads, int kv_heads, int head_dim,
                                             int table_width, int page_size, int64_t* bytes) {
  QIE_CHECK_ARG(bytes && tokens >= 0 && seqs > 0 && heads > 0 && kv_heads > 0 && head_dim > 0 && table_width > 0 &&
                page_size > 0 && (int64_t)table_width * page_size <= INT32_MAX / 2);
  const SeqPlan p = seq_plan(tokens, seqs, heads, kv_heads, head_dim, true, (int64_t)table_width * page_size);
  *bytes = p.ct ? (int64_t)tokens * heads * p.maxch * (head_dim + 2) * 4
                : (int64_t)p.shares * 2 * kv_heads * kPPRows * (head_dim + 2) * 4;
  return QIE_OK;
}

extern "C" int qie_attention_paged_bf16(const void* q, int64_t ldq, int64_t hsq, const void* k_pages,
                                        const void* v_pages, int num_pages, int page_size, int64_t page_stride,
                                        int64_t page_head_stride, int64_t slot_stride, const int* page_table,
                                        int64_t ld_table, int table_width, const int* kv_lens, const int* cu_seqlens,
                                        int seqs, int tokens, int heads, int kv_heads, int head_dim, float scale,
                                        void* out, int64_t ldo, int64_t hso, void* workspace, int64_t workspace_bytes,
                                        qie_stream_t stream) {
  QIE_CHECK_ARG(seq_common_ok(q, ldq, hsq, k_pages, v_pages, slot_stride, page_head_stride, seqs, tokens, heads,
                              kv_heads, head_dim, scale, out, ldo, hso));
  QIE_CHECK_ARG(page_table && kv_lens && (cu_seqlens || seqs == tokens) && num_pages > 0 && table_width > 0);
  QIE_CHECK_ARG(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0);
  QIE_CHECK_ARG(page_stride >= 0 && page_stride % 8 == 0 && (ld_table >= table_width || ld_table == 0));
  QIE_CHECK_ARG((int64_t)table_width * page_size <= INT32_MAX / 2);
  int64_t need = 0;
  const int rc = qie_attention_paged_workspace(tokens, seqs, heads, kv_heads, head_dim, table_width, page_size, &need);
  if (rc) return rc;
  QIE_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0));
  if (tokens == 0) return QIE_OK;
  SeqArgs a{};
  a.q = (const bf16_t*)q; a.ldq = ldq; a.hsq = hsq;
  a.k = (const bf16_t*)k_pages; a.v = (const bf16_t*)v_pages; a.ldk = slot_stride; a.hsk = page_head_stride;
  a.out = (bf16_t*)out; a.ldo = ldo; a.hso = hso;
  a.cu = cu_seqlens;
  a.B = seqs; a.T = tokens; a.H = heads; a.Hk = kv_heads; a.G = heads / kv_heads; a.Dh = head_dim;
  a.causal = 1;
  set_scale(a, scale);
  a.table = page_table; a.ldt = ld_table; a.ps = page_stride;
  a.kv_lens = kv_lens;
  a.width = table_width; a.pages = num_pages; a.pshift = __builtin_ctz(page_size);
  a.ws = (float*)workspace;
  return launch_seq(a, seq_plan(tokens, seqs, heads, kv_heads, head_dim, true, (int64_t)table_width * page_size), true,
                    (hipStream_t)stream);
}
