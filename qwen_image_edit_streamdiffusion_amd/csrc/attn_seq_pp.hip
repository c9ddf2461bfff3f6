// Attention over sequences for many rows: one work-group = 8 waves = 256 rows (tokens x the G query
// heads of one kv head) of one sequence, 32 rows a wave, 64-key tiles. The products are those of
// attn_seq.hip on mfma 32x32x16 (S^T = K Q^T, O^T += V^T P^T; a lane holds 32 keys of one row).
//
// Waves 0-3 and 4-7 put one wave of each group on every SIMD, one phase apart: while one is in its matrix phase
// (S of tile t, then O += V P of tile t - 1, operands read from LDS six products ahead) the other is in its
// softmax phase. K and V live in 4-slot LDS rings; softmax phase t issues the LDS-DMA of K(t + 3) and
// V(t + 2) and ends when what it issued a phase earlier has landed, so every tile is there two
// phases before its first read and one barrier ends each phase. The products are asm volatile:
// their order and the LDS reads between them stay as written; register fences pin the softmax
// inside its phase. Measured (device, median), 28 heads of 128 over 4: four causal sequences of up to 8192 690 .. 745 us
// on one card and another (1095 .. 1015 TFLOP/s), 32768 causal rows 6.4 .. 6.7 ms (1200 .. 1150), chunks of 300 .. 1500
// tokens over 5000 .. 24000 cached keys 505 .. 520 and 20 for the join. A tile of 128-wide heads takes a CU 3450 cycles
// (paged: 4110): the matrix pipe of a SIMD is busy for 2048 of them, the other wave's 250 vector instructions take
// about as many, no LDS bank conflicts. So neither unit is the bound; the phases take 1.7 times the longer of the two
// (paged: 2), and what they wait for in between has not been separated.
#include <type_traits>

#include "attn_seq.h"

namespace {

constexpr int kRing = 4;

__device__ __forceinline__ void mma32(f32x16_t& c, const bf16x8_t& a, const bf16x8_t& b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mma32_z(f32x16_t& c, const bf16x8_t& a, const bf16x8_t& b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}
template <typename T>
__device__ __forceinline__ void rfence(T& x) {
  asm volatile("" : "+v"(x));
}

// ---- Shares: blocks that do not fill the chip, or not evenly, are cut where the work is, not at a fixed
// count of keys. The blocks of one kv head lie behind each other on a line, each as long as the keys that it
// sees; work-group s of a.shares takes the s-th equal part: the end of one block, whole blocks, the
// beginning of another. Only the first and the last leave fp32 parts (m, l, O), two slots a work-group,
// and a second kernel joins them. Lengths are device memory, so the line is laid out here, by every wave.
constexpr int kUnit = 16;              // keys of a unit of the line: sums over all blocks stay in 32 bits (the host sees to it)
constexpr int kShare = 512 / kUnit;    // fewest units of a share
constexpr int kBlockKeys = 160;        // what beginning and ending a block costs, in keys
constexpr int kCut = 1800 / kUnit;     // what cuts cost a call: parts written and read, the join (50 us)

struct Line {  // a block of the line: sequence, its place on the line, the block's ends there
  int b, start, n, kv, nblk, blk;
  int base, c0, c1;
};
// where block x of a sequence begins: the sum of (cost + kept + 256 (i + 1) / G) over the blocks before it
__device__ __forceinline__ int line_at(const SeqArgs& a, int n, int kv, int x) {
  const int64_t keys = (int64_t)x * (max(kv - n, 0) + kBlockKeys) + (int64_t)((double)((int64_t)(kPPRows / 2) * x * (x + 1)) / a.G);
  return (int)(keys / kUnit);
}
struct LineSeq {  // a lane's sequence: length on the line, blocks
  int start, n, kv, nblk, c;
};
__device__ __forceinline__ LineSeq line_seq(const SeqArgs& a, int b) {
  LineSeq s{0, 0, 0, 0, 0};
  if (b < a.B) {
    seq_span<true>(a, b, s.start, s.n, s.kv);
    s.nblk = (s.n * a.G + kPPRows - 1) / kPPRows;
    s.c = line_at(a, s.n, s.kv, s.nblk);
  }
  return s;
}
// The line's length and how it is cut: ns equal shares; or, where no block is much longer than a share would
// be, whole blocks (8 x 200 new tokens over 5000 keys: 151 us, 157 in shares; 16 x 100: level at 165)
struct Cuts {
  int total, ns;
  bool whole;
};
__device__ __forceinline__ Cuts line_cuts(const SeqArgs& a, LineSeq& first) {
  const int lane = threadIdx.x & 63;
  int v = 0, blocks = 0, longest = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const LineSeq s = line_seq(a, b0 + lane);
    if (b0 == 0) first = s;
    v += s.c;
    blocks += s.nblk;
    if (s.nblk) longest = max(longest, s.c - line_at(a, s.n, s.kv, s.nblk - 1));
  }
  Cuts c;
  c.total = __builtin_amdgcn_readlane(wave_scan(v), 63);
  blocks = __builtin_amdgcn_readlane(wave_scan(blocks), 63);
  longest = (int)wave_max((float)longest);
  c.ns = min(a.shares, max(1, c.total / kShare));
  c.whole = blocks <= a.shares && uni(longest) <= c.total / c.ns + kCut;
  if (c.whole) c.ns = blocks;
  return c;
}
__device__ __forceinline__ void line_block(const SeqArgs& a, Line& l, int x) {
  l.blk = x;
  l.c0 = l.base + line_at(a, l.n, l.kv, x);
  l.c1 = l.base + line_at(a, l.n, l.kv, x + 1);
}
// the block that holds position at (< the line's length), or block number at; first: line_cuts' lanes.
// false: none, as where offsets overlap and the sums pass 32 bits
__device__ __forceinline__ bool line_seek(const SeqArgs& a, const LineSeq& first, int at, Line& l, bool number = false) {
  const int lane = threadIdx.x & 63;
  l.base = l.nblk = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const LineSeq s = b0 == 0 ? first : line_seq(a, b0 + lane);
    const int c = number ? s.nblk : s.c, pre = wave_scan(c);
    const unsigned long long hit = __ballot(l.base + pre > at);
    if (hit) {
      const int i = __builtin_ctzll(hit);
      l.b = b0 + i;
      l.start = __builtin_amdgcn_readlane(s.start, i);
      l.n = __builtin_amdgcn_readlane(s.n, i);
      l.kv = __builtin_amdgcn_readlane(s.kv, i);
      l.nblk = __builtin_amdgcn_readlane(s.nblk, i);
      l.base += __builtin_amdgcn_readlane(pre - c, i);
      break;
    }
    l.base += __builtin_amdgcn_readlane(pre, 63);
  }
  if (l.nblk <= 0) return false;
  if (number) {
    const int x = min(max(at - l.base, 0), l.nblk - 1);
    l.base = 0;
    line_block(a, l, x);
    return true;
  }
  int lo = 0, hi = l.nblk - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.base + line_at(a, l.n, l.kv, mid) <= at) lo = mid;
    else hi = mid - 1;
  }
  line_block(a, l, lo);
  return true;
}
__device__ __forceinline__ bool line_next(const SeqArgs& a, Line& l) {
  if (l.blk + 1 < l.nblk) {
    line_block(a, l, l.blk + 1);
    return true;
  }
  l.base = l.c1;
  for (++l.b; l.b < a.B; ++l.b) {
    seq_span<true>(a, l.b, l.start, l.n, l.kv);
    if (l.n == 0) continue;
    l.nblk = (l.n * a.G + kPPRows - 1) / kPPRows;
    line_block(a, l, 0);
    return true;
  }
  return false;
}
// 64-key tiles of a block; the tile at which position at cuts it
__device__ __forceinline__ int line_tiles(const SeqArgs& a, const Line& l) {
  const int last = (min(l.n * a.G, (l.blk + 1) * kPPRows) - 1) / a.G;
  return (min(l.kv, max(l.kv - l.n + last + 1, 0)) + kKB - 1) / kKB;
}
__device__ __forceinline__ int line_tile(const Line& l, int at, int ntot) {
  if (at <= l.c0) return 0;
  return at >= l.c1 ? ntot : (int)((double)(at - l.c0) * ntot / (double)(l.c1 - l.c0));
}
// where share i of ns begins
__device__ __forceinline__ int share_cut(int total, int ns, int i) { return (int)((double)total * i / ns); }
// the fp32 part of work-group sh that begins its block (first) or goes on with it
__device__ __forceinline__ float* share_part(const SeqArgs& a, int sh, bool first, int hk) {
  return a.ws + ((int64_t)(2 * sh + first) * a.Hk + hk) * kPPRows * (a.Dh + 2);
}

template <bool SHARE, bool PAGED, int KS>  // KS 16-wide steps of the head (4, 6, 8): head_dim <= 16 KS
__global__ void __launch_bounds__(512) attn_seq_pp_kernel(SeqArgs args) {
  constexpr int ND = KS / 2;  // 32-wide blocks of the output
  constexpr int NQ = 2 * KS, NP = 4 * ND;
  __shared__ __attribute__((aligned(16))) char smem_raw[2 * kRing * kTile];  // K ring, V ring
  char QIE_LDS* smem = (char QIE_LDS*)smem_raw;

  Item it;
  // between two blocks of a share its place waits here: in scalar registers it would push the tiles'
  // addresses out of them
  __shared__ struct { Line line, head; int end, head_t0; } place;
  int t0 = 0;
  bool tail = false;
  if constexpr (SHARE) {
    const SeqArgs& a = args;
    const int sh = blockIdx.x / a.Hk;
    LineSeq first;
    const Cuts cuts = line_cuts(a, first);
    if (sh >= cuts.ns) return;
    int begin = share_cut(cuts.total, cuts.ns, sh), end = share_cut(cuts.total, cuts.ns, sh + 1);
    if (!cuts.whole && begin >= end) return;
    Line head, line;
    if (!line_seek(a, first, cuts.whole ? sh : begin, head, cuts.whole)) return;
    if (cuts.whole) {
      begin = head.c0;
      end = head.c1;
    }
    line = head;
    t0 = line_tile(head, begin, line_tiles(a, head));
    const int head_t0 = t0;
    if (!cuts.whole && end < cuts.total) {
      // the beginning of the last block goes first: its tiles and then the first block's are those that the other
      // work-groups of the sequence read at the same time (L2)
      Line l;
      if (line_seek(a, first, end, l) && l.c0 > begin && line_tile(l, end, line_tiles(a, l)) > 0) {
        line = l;
        tail = true;
        t0 = 0;
      }
    }
    if (threadIdx.x == 0) {
      place.line = line;
      place.head = head;
      place.end = end;
      place.head_t0 = head_t0;
    }
    __syncthreads();
  } else {
    if (!find_item<PAGED, kPPRows>(args, blockIdx.x / args.Hk, it)) return;
  }
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int grp = wave >> 2, hf = lane >> 5, ql = lane & 31;
  for (;;) {
  // a share's next block reads the arguments anew: kept over the blocks they would fill the scalar registers
  auto fresh = [&]() -> SeqArgs {
    if constexpr (!SHARE) return args;
    typedef const uint32_t __attribute__((address_space(4))) Word;
    Word* p = (Word*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    struct { uint32_t w[sizeof(SeqArgs) / 4]; } raw;
#pragma unroll
    for (unsigned i = 0; i < sizeof(SeqArgs) / 4; ++i) raw.w[i] = p[i];
    return __builtin_bit_cast(SeqArgs, raw);
  };
  const SeqArgs a = fresh();
  const int hk = blockIdx.x % a.Hk;
  if constexpr (SHARE) {
    it.b = uni(place.line.b); it.start = uni(place.line.start); it.n = uni(place.line.n); it.kv = uni(place.line.kv);
    it.blk = uni(place.line.blk);
  }
  const int rows = it.n * a.G;
  const int r = it.blk * kPPRows + wave * 32 + ql;
  const int rc = min(r, rows - 1);
  const int tok = rc / a.G, head = hk * a.G + rc % a.G;
  const int off = it.kv - it.n;
  const int lim = a.causal ? min(it.kv, max(off + tok + 1, 0)) : it.kv;  // keys that this row sees
  const int lim0 = uni(lim);                                             // fewest of the wave
  const int last = (min(rows, (it.blk + 1) * kPPRows) - 1) / a.G;
  const int most = a.causal ? min(it.kv, max(off + last + 1, 0)) : it.kv;
  const int ntot = (most + kKB - 1) / kKB;
  int ntiles = ntot;
  if constexpr (SHARE) {
    ntiles = uni(line_tile(place.line, place.end, ntot));
  } else if (PAGED && a.ct) {
    t0 = it.ch * a.ct;
    if (t0 > 0 && t0 >= ntot) return;  // a causal block that ends before this chunk
    ntiles = min(ntot, t0 + a.ct);
  }
  const bool whole = SHARE ? t0 == 0 && ntiles == ntot : !PAGED || !a.ct || ntot <= a.ct;

  bf16x8_t qf[KS];
  f32x16_t s[2], o[ND];
  bf16x8_t pf[4];
  float m_run = a.low, l_run = 0.f;
  float above = kRescale, mscale = a.c;  // seq_far
#pragma unroll
  for (int db = 0; db < ND; ++db) o[db] = f32x16_t{};

  // ---- LDS-DMA: wave w fills rows 4(w + 8p) .. +3 of a tile (p = 0, 1) of K and of V; the lane's
  // source chunk carries the XOR swizzle. What lies past the head or the sequence arrives as zeros.
  const uint32_t ldb = (uint32_t)(a.ldk * 2);
  uint32_t ko[2], vo[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = (wave + 8 * p) * 4 + (lane >> 4), c = lane & 15;
    const int ck = c ^ (row & 15), cv = c ^ ((row & 3) << 2);
    // packed rows: offsets within the tile; pages: within the 4-row piece
    const uint32_t ro = (PAGED ? (uint32_t)(lane >> 4) : (uint32_t)row) * ldb;
    ko[p] = ck * 8 < a.Dh ? ro + ck * 16 : 0x80000000u;
    vo[p] = cv * 8 < a.Dh ? ro + cv * 16 : 0x80000000u;
  }
  const int head_bytes = a.Dh * 2;
  const char* kbase = (const char*)(a.k + (int64_t)hk * a.hsk) + (PAGED ? 0 : (int64_t)it.start * ldb);
  const char* vbase = (const char*)(a.v + (int64_t)hk * a.hsk) + (PAGED ? 0 : (int64_t)it.start * ldb);
  // pages: lane i holds the page of tile tb + i's piece p (-1: outside the pool)
  const int* table = PAGED ? a.table + (int64_t)it.b * a.ldt : nullptr;
  int tb = 0, pg[2] = {0, 0};
  auto pages = [&](int from) {
    tb = from;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int key = (from + lane) * kKB + (wave + 8 * p) * 4;
      int id = -1;
      if (key < it.kv) id = table[key >> a.pshift];
      pg[p] = id >= 0 && id < a.pages ? id : -1;
    }
  };
  auto dma1 = [&](const char* base, const uint32_t (&vo_)[2], int t, int ring) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int r0 = (wave + 8 * p) * 4;
      i32x4_t rs;
      if constexpr (PAGED) {
        const int key = t * kKB + r0, nrow = min(4, it.kv - key);
        const int id = __builtin_amdgcn_readlane(pg[p], t - tb);
        const bool ok = nrow > 0 && id >= 0;
        const int64_t at = ok ? ((int64_t)id * a.ps + (int64_t)(key & ((1 << a.pshift) - 1)) * a.ldk) * 2 : 0;
        rs = seq_rsrc((const bf16_t*)(base + at), ok ? (nrow - 1) * (int)ldb + head_bytes : 0);
      } else {
        const int nrow = min(kKB, it.kv - t * kKB);
        rs = seq_rsrc((const bf16_t*)(base + (int64_t)t * kKB * ldb), (nrow - 1) * (int)ldb + head_bytes);
      }
      seq_dma(rs, smem + (ring * kRing + (t & (kRing - 1))) * kTile + r0 * kRowB, vo_[p]);
    }
  };
  auto dmaK = [&](int t) { dma1(kbase, ko, t, 0); };
  auto dmaV = [&](int t) { dma1(vbase, vo, t, 1); };

  const int ksw = lane & 15;
  const int tr_row = (lane & 15) >> 2, tr_sw = tr_row << 2, tr_g1 = (lane >> 4) & 1, tr_cb = 8 * (lane & 1);
  auto kfrag = [&](int cb, int ks, int t) -> bf16x8_t {
    const char QIE_LDS* krow = smem + (t & (kRing - 1)) * kTile + (cb * 32 + ql) * kRowB;
    return *(const bf16x8_t QIE_LDS*)(krow + (((2 * ks + hf) ^ ksw) << 4));
  };
  // V^T: lane's d = 32 db + ql, keys 16 ks + 4 hf + 0..3 and 8 further
  auto vfrag = [&](int ks, int db, int t) -> bf16x8_t {
    const char QIE_LDS* vb = smem + (kRing + (t & (kRing - 1))) * kTile;
    const int chunk = (4 * db + 2 * tr_g1 + ((lane & 3) >> 1)) ^ tr_sw;
    const char QIE_LDS* p0 = vb + (16 * ks + 4 * hf + tr_row) * kRowB + (chunk << 4) + tr_cb;
    const s16x4_t va = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t QIE_LDS*)p0);
    const s16x4_t vb2 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t QIE_LDS*)(p0 + 8 * kRowB));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(va, vb2, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // product i of a matrix phase: i < NQ the S^T chain of tile tk, then O^T += V^T P^T of tile tv
  auto opA = [&](int i, int tk, int tv) -> bf16x8_t {
    if (i < NQ) return kfrag(i / KS, i % KS, tk);
    return vfrag((i - NQ) / ND, (i - NQ) % ND, tv);
  };
  auto mfma_i = [&](int i, const bf16x8_t& A) {
    if (i < NQ) {
      if (i % KS == 0) mma32_z(s[i / KS], A, qf[0]);
      else mma32(s[i / KS], A, qf[i % KS]);
    } else {
      mma32(o[(i - NQ) % ND], A, pf[(i - NQ) / ND]);
    }
  };
  constexpr int PF = 6;  // operand prefetch distance in products
  bf16x8_t A[8];
  // products [i0, i1) with the operands up to i2 (the next part's first ones) read on the way
  auto products = [&](auto i0_t, auto i1_t, auto i2_t, int tk, int tv) {
    constexpr int i0 = decltype(i0_t)::value, i1 = decltype(i1_t)::value, i2 = decltype(i2_t)::value;
#pragma unroll
    for (int i = i0; i < i1; ++i) {
      if (i + PF < i2) A[(i + PF) & 7] = opA(i + PF, tk, tv);
      mfma_i(i, A[i & 7]);
    }
  };
  auto first = [&](auto i0_t, int tk, int tv) {
    constexpr int i0 = decltype(i0_t)::value;
#pragma unroll
    for (int i = i0; i < i0 + PF; ++i) A[i & 7] = opA(i, tk, tv);
  };
  bool done = false;  // this tile's O += V P is done already (masked infinities or NaN)
  auto vphase = [&](int t) {
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) rfence(s[cb]);
#pragma unroll
    for (int db = 0; db < ND; ++db) rfence(o[db]);
    int pieces = 0;
    if constexpr (PAGED)
      if (t + 3 < ntiles && t + 3 - tb >= 64) {
        pages(t + 2);
        __builtin_amdgcn_s_waitcnt(0);
      }
    if (t + 3 < ntiles) { dmaK(t + 3); pieces += 2; }
    if (t + 2 < ntiles) { dmaV(t + 2); pieces += 2; }
    const int kv0 = t * kKB;
    const bool masked = kv0 + kKB > lim0;
    if (masked) {
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kv0 + cb * 32 + (i & 3) + 8 * (i >> 2) + 4 * hf >= lim) s[cb][i] = -INFINITY;
    }
    float m0 = fmaxf(s[0][0], s[0][1]), m1 = fmaxf(s[0][2], s[0][3]);
#pragma unroll
    for (int i = 4; i < 16; i += 2) { m0 = fmaxf(m0, s[0][i]); m1 = fmaxf(m1, s[0][i + 1]); }
#pragma unroll
    for (int i = 0; i < 16; i += 2) { m0 = fmaxf(m0, s[1][i]); m1 = fmaxf(m1, s[1][i + 1]); }
    float mx = fmaxf(m0, m1);
    {  // with the row's other half-wave
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    }
    if (__any((mx - m_run) * a.c > above)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * a.c);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < ND; ++db) o[db] *= alpha;
      if (__builtin_expect(seq_far(a, m_run, above, mscale), 0))
#pragma unroll
        for (int i = 0; i < 32; ++i) s[i >> 4][i & 15] -= m_run;
    }
    const float mc = m_run * mscale;
    float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cb][i], a.c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cb][i + 1], a.c, -mc));
        ps0 += p0;
        ps1 += p1;
        pf[cb * 2 + (i >> 3)][i & 7] = (__bf16)p0;
        pf[cb * 2 + (i >> 3)][(i & 7) + 1] = (__bf16)p1;
      }
    l_run += ps0 + ps1;
    done = false;
    if (masked) {  // V(t) landed a phase ago: are there infinities or NaN that a row must not see?
      Magnitude mag;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
        for (int db = 0; db < ND; ++db) mag.add(vfrag(ks, db, t));
        asm volatile("" ::: "memory");  // few fragments in registers at a time
      }
      if (__builtin_expect(__any(mag.nonfinite()), 0)) {
        done = true;  // O += V P here: the finite values, then what a row sees of the others
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          bf16x8_t fin = finite(vfrag(j / ND, j % ND, t));
          asm volatile("s_nop 4" : "+v"(fin)::"memory");
          mma32(o[j % ND], fin, pf[j / ND]);
        }
#pragma unroll
        for (int db = 0; db < ND; ++db) asm volatile("s_nop 15\n\ts_nop 7" : "+v"(o[db]));
#pragma unroll 1
        for (int j = 0; j < kKB; ++j) {
          const char QIE_LDS* vr = smem + (kRing + (t & (kRing - 1))) * kTile + j * kRowB + 8 * hf;
          const bool see = kv0 + j < lim;
#pragma unroll
          for (int db = 0; db < ND; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const u32x2_t w = *(const u32x2_t QIE_LDS*)(vr + (((4 * db + g) ^ ((j & 3) << 2)) << 4));
#pragma unroll
              for (int i = 0; i < 4; ++i) o[db][4 * g + i] += special(i < 2 ? w.x : w.y, i & 1, see);
            }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) rfence(pf[k]);
    rfence(l_run);
    rfence(m_run);
#pragma unroll
    for (int db = 0; db < ND; ++db) rfence(o[db]);
    if (pieces == 4) asm volatile("s_waitcnt vmcnt(4)\n\ts_barrier" ::: "memory");
    else if (pieces == 2) asm volatile("s_waitcnt vmcnt(2)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  };
  using I0 = std::integral_constant<int, 0>;
  using IQ = std::integral_constant<int, NQ>;
  using IA = std::integral_constant<int, NQ + NP>;

  if (t0 < ntiles) {
    if constexpr (PAGED) {
      pages(t0);
      __builtin_amdgcn_s_waitcnt(0);
    }
    // K(t0 .. t0 + 2), V(t0), V(t0 + 1) resident; group 1 waits one phase
    dmaK(t0);
    if (t0 + 1 < ntiles) dmaK(t0 + 1);
    dmaV(t0);
    if (t0 + 2 < ntiles) dmaK(t0 + 2);
    if (t0 + 1 < ntiles) dmaV(t0 + 1);
    {
      const bf16_t* qr = a.q + (int64_t)(it.start + tok) * a.ldq + (int64_t)head * a.hsq + 8 * hf;
  #pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = bf16x8_t{};
        if (16 * ks + 8 * hf < a.Dh) qf[ks] = *(const bf16x8_t*)(qr + 16 * ks);
      }
    }
    __builtin_amdgcn_s_waitcnt(0);  // q as well: from here on the counter is the tiles'
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    if (grp == 1) asm volatile("s_barrier" ::: "memory");
    // asm products are not padded: the softmax may read the last ones' results (S on the first tile) 16 cycles on
    auto mend = [&]() { asm volatile("s_nop 15\n\ts_barrier" ::: "memory"); };
    first(I0{}, t0, t0);
    products(I0{}, IQ{}, IQ{}, t0, t0);
    mend();
    vphase(t0);
    for (int t = t0 + 1; t < ntiles; ++t) {
      __builtin_amdgcn_s_setprio(2);  // over the SIMD's other wave, in its softmax phase
      first(I0{}, t, t - 1);
      products(I0{}, IQ{}, IA{}, t, t - 1);                 // S(t)
      if (!done) products(IQ{}, IA{}, IA{}, t, t - 1);      // O += V(t - 1) P(t - 1)
      __builtin_amdgcn_s_setprio(0);
      mend();
      vphase(t);
    }
    if (!done) {
      first(IQ{}, t0, ntiles - 1);
      products(IQ{}, IA{}, IA{}, t0, ntiles - 1);
    }
    if (grp == 0) asm volatile("s_barrier" ::: "memory");
    // asm products are not padded: their results are read next
#pragma unroll
    for (int db = 0; db < ND; ++db) asm volatile("s_nop 15\n\ts_nop 7" : "+v"(o[db]));
  }
  const SeqArgs e = fresh();
  const float l = l_run + __shfl_xor(l_run, 32, 64);
  if (r < rows && !whole && t0 < ntiles) {
    const int br = wave * 32 + ql;  // row of the block
    float *po, *pml;
    if constexpr (SHARE) {
      float* part = share_part(e, blockIdx.x / e.Hk, t0 == 0, hk);
      po = part + br * e.Dh;
      pml = part + kPPRows * e.Dh + 2 * br;
    } else {
      const int64_t pi = ((int64_t)(it.start + tok) * e.H + head) * e.maxch + it.ch;
      po = e.ws + pi * e.Dh;
      pml = e.ws + (int64_t)e.T * e.H * e.maxch * e.Dh + pi * 2;
    }
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * db + 8 * g < e.Dh)
          *(f32x4_t*)(po + 32 * db + 8 * g + 4 * hf) =
              f32x4_t{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    if (hf == 0) *(f32x2_t*)pml = f32x2_t{m_run, l};
  }
  if (r < rows && whole) {
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key seen: o is 0 as well
  bf16_t* dst = e.out + (int64_t)(it.start + tok) * e.ldo + (int64_t)head * e.hso;
  // lane (ql, hf) holds d = 32 db + 8 g + 4 hf + 0..3; a swap of halves for two g gives 16-byte stores
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      const uint32_t w0 = pack2(o[db][4 * g] * inv, o[db][4 * g + 1] * inv);
      const uint32_t w1 = pack2(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv);
      const uint32_t w2 = pack2(o[db][4 * g + 4] * inv, o[db][4 * g + 5] * inv);
      const uint32_t w3 = pack2(o[db][4 * g + 6] * inv, o[db][4 * g + 7] * inv);
      const auto sx = __builtin_amdgcn_permlane32_swap(w0, w2, false, false);
      const auto sy = __builtin_amdgcn_permlane32_swap(w1, w3, false, false);
      if (32 * db + 8 * g + 8 * hf < e.Dh)
        *(u32x4_t*)(dst + 32 * db + 8 * g + 8 * hf) = u32x4_t{sx[0], sy[0], sx[1], sy[1]};
    }
  }
  if constexpr (!SHARE) return;
  Line line = place.line;
  int end = place.end;
  bool more = true;
  if (tail) {
    end = line.c0;
    line = place.head;
    t0 = uni(place.head_t0);
    tail = false;
  } else {
    more = line.c1 < end && line_next(e, line);
    t0 = 0;
  }
  __syncthreads();  // the rings are free, the place is read
  if (!more) return;
  if (threadIdx.x == 0) {
    place.line = line;
    place.end = end;
  }
  __syncthreads();
  }
}

// Joins a block's parts: o = sum_p w_p o_p / sum_p w_p l_p, w_p = exp2((m_p - max m) c). Work-groups
// [kJoinSplit (s - 1), ..) of a kv head look at the cut between shares s - 1 and s and join the block that it
// cuts first; a wave eight rows, two elements a lane.
constexpr int kJoinRows = 8, kJoinSplit = kPPRows / (4 * kJoinRows);
__global__ void __launch_bounds__(256) attn_seq_join_shares_kernel(SeqArgs a) {
  const int hk = blockIdx.x % a.Hk, u = blockIdx.x / a.Hk, s = 1 + u / kJoinSplit;
  LineSeq first;
  const Cuts cuts = line_cuts(a, first);
  const int ns = cuts.ns;
  if (cuts.whole || s >= ns) return;
  auto cut = [&](int i) { return share_cut(cuts.total, ns, i); };
  Line l;
  if (!line_seek(a, first, cut(s), l)) return;
  const int ntot = line_tiles(a, l), t = line_tile(l, cut(s), ntot);
  if (t == 0 || t == ntot || line_tile(l, cut(s - 1), ntot) > 0) return;
  const int lane = threadIdx.x & 63, d = 2 * lane < a.Dh ? 2 * lane : 0;
  const int rows = min(kPPRows, l.n * a.G - l.blk * kPPRows);
  const int br = kJoinRows * (4 * (u % kJoinSplit) + uni(threadIdx.x >> 6));  // rows br ..
  if (br >= rows) return;
  float m[kJoinRows], L[kJoinRows], o0[kJoinRows], o1[kJoinRows];
#pragma unroll
  for (int j = 0; j < kJoinRows; ++j) {
    m[j] = a.low;
    L[j] = o0[j] = o1[j] = 0.f;
  }
  for (int i0 = s - 1; i0 < ns && cut(i0) < l.c1; i0 += 64) {
    const int me = i0 + lane;  // a lane looks whether its share left a part
    const bool has = me < ns && cut(me) < l.c1 && (me < s || line_tile(l, cut(me), ntot) < line_tile(l, cut(me + 1), ntot));
    for (unsigned long long left = __ballot(has); left; left &= left - 1) {
      const int i = i0 + __builtin_ctzll(left);
      const float* p = share_part(a, i, i < s, hk);
      f32x2_t ml[kJoinRows], v[kJoinRows];
#pragma unroll
      for (int j = 0; j < kJoinRows; ++j) {  // rows past the block's last: their part is there, and unread below
        ml[j] = *(const f32x2_t*)(p + kPPRows * a.Dh + 2 * (br + j));
        v[j] = *(const f32x2_t*)(p + (br + j) * a.Dh + d);
      }
#pragma unroll
      for (int j = 0; j < kJoinRows; ++j) {
        const float mn = fmaxf(m[j], ml[j][0]);
        const float f = __builtin_amdgcn_exp2f((m[j] - mn) * a.c), w = __builtin_amdgcn_exp2f((ml[j][0] - mn) * a.c);
        m[j] = mn;
        L[j] = __builtin_fmaf(w, ml[j][1], L[j] * f);
        o0[j] = __builtin_fmaf(w, v[j][0], o0[j] * f);
        o1[j] = __builtin_fmaf(w, v[j][1], o1[j] * f);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kJoinRows; ++j) {
    const float inv = L[j] == 0.f ? 0.f : 1.0f / L[j];
    const int r = l.blk * kPPRows + br + j, tok = r / a.G, head = hk * a.G + r % a.G;
    if (br + j < rows && 2 * lane < a.Dh)
      *(uint32_t*)(a.out + (int64_t)(l.start + tok) * a.ldo + (int64_t)head * a.hso + d) = pack2(o0[j] * inv, o1[j] * inv);
  }
}

template <bool SHARE, bool PAGED>
int launch(const SeqArgs& a, unsigned grid, hipStream_t s) {
  if (a.Dh <= 64) attn_seq_pp_kernel<SHARE, PAGED, 4><<<grid, 512, 0, s>>>(a);
  else if (a.Dh <= 96) attn_seq_pp_kernel<SHARE, PAGED, 6><<<grid, 512, 0, s>>>(a);
  else attn_seq_pp_kernel<SHARE, PAGED, 8><<<grid, 512, 0, s>>>(a);
  return qie_last_error();
}

}  // namespace

int qie_launch_seq_pp(const SeqArgs& a, bool paged, hipStream_t s) {
  const int64_t rb = (int64_t)a.T * a.G / kPPRows + a.B;  // at least the row blocks of any lengths
  const int64_t grid = rb * a.maxch * a.Hk;
  if (grid > INT32_MAX || (int64_t)a.shares * a.Hk * kJoinSplit > INT32_MAX) return QIE_ERR_UNSUPPORTED;
  if (!a.shares) return paged ? launch<false, true>(a, (unsigned)grid, s) : launch<false, false>(a, (unsigned)grid, s);
  const int rc = launch<true, true>(a, (unsigned)(a.shares * a.Hk), s);
  if (rc || a.shares == 1) return rc;
  attn_seq_join_shares_kernel<<<(unsigned)((a.shares - 1) * a.Hk * kJoinSplit), 256, 0, s>>>(a);
  return qie_last_error();
}
