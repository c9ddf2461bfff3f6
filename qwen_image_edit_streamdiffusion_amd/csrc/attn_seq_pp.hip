// Attention over sequences for many rows: one work-group = 8 waves = 256 rows (tokens x the G query
// heads of one kv head) of one sequence, 32 rows a wave, 64-key tiles. The products are those of
// attn_seq.hip on mfma 32x32x16 (S^T = K Q^T, O^T += V^T P^T; a lane holds 32 keys of one row).
//
// Bound by the matrix pipe and, beside it, by the softmax's vector issue. Waves 0-3 and 4-7 put one
// wave of each group on every SIMD, one phase apart: while one is in its matrix phase (S of tile t,
// then O += V P of tile t - 1, operands read from LDS five products ahead) the other is in its
// softmax phase. K and V live in 4-slot LDS rings; softmax phase t issues the LDS-DMA of K(t + 3) and
// V(t + 2) and ends when what it issued a phase earlier has landed, so every tile is there two
// phases before its first read and one barrier ends each phase. The products are asm volatile:
// their order and the LDS reads between them stay as written; register fences pin the softmax
// inside its phase.
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

template <bool PAGED, int KS>  // KS 16-wide steps of the head (4, 6, 8): head_dim <= 16 KS
__global__ void __launch_bounds__(512) attn_seq_pp_kernel(SeqArgs a) {
  constexpr int ND = KS / 2;  // 32-wide blocks of the output
  constexpr int NQ = 2 * KS, NP = 4 * ND;
  __shared__ __attribute__((aligned(16))) char smem_raw[2 * kRing * kTile];  // K ring, V ring
  char QIE_LDS* smem = (char QIE_LDS*)smem_raw;

  const int hk = blockIdx.x % a.Hk;
  Item it;
  if (!find_item<PAGED, kPPRows>(a, blockIdx.x / a.Hk, it)) return;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int grp = wave >> 2, hf = lane >> 5, ql = lane & 31;
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
  const int t0 = a.ct ? it.ch * a.ct : 0;
  const int ntiles = a.ct ? min(ntot, t0 + a.ct) : ntot;
  const bool whole = !a.ct || ntot <= a.ct;
  if (t0 > 0 && t0 >= ntot) return;  // a causal block that ends before this chunk

  bf16x8_t qf[KS];
  f32x16_t s[2], o[ND];
  bf16x8_t pf[4];
  float m_run = kLow, l_run = 0.f;
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
  constexpr int PF = 5;  // operand prefetch distance in products
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
    if (__any((mx - m_run) * a.c > kRescale)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * a.c);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < ND; ++db) o[db] *= alpha;
    }
    const float mc = m_run * a.c;
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
  const float l = l_run + __shfl_xor(l_run, 32, 64);
  if (r >= rows) return;
  if (!whole) {
    const int64_t pi = ((int64_t)(it.start + tok) * a.H + head) * a.maxch + it.ch;
    float* po = a.ws + pi * a.Dh;
    float* pml = a.ws + (int64_t)a.T * a.H * a.maxch * a.Dh + pi * 2;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * db + 8 * g < a.Dh)
          *(f32x4_t*)(po + 32 * db + 8 * g + 4 * hf) =
              f32x4_t{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    if (hf == 0) *(f32x2_t*)pml = f32x2_t{m_run, l};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key seen: o is 0 as well
  bf16_t* dst = a.out + (int64_t)(it.start + tok) * a.ldo + (int64_t)head * a.hso;
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
      if (32 * db + 8 * g + 8 * hf < a.Dh)
        *(u32x4_t*)(dst + 32 * db + 8 * g + 8 * hf) = u32x4_t{sx[0], sy[0], sx[1], sy[1]};
    }
}

template <bool PAGED>
int launch(const SeqArgs& a, unsigned grid, hipStream_t s) {
  if (a.Dh <= 64) attn_seq_pp_kernel<PAGED, 4><<<grid, 512, 0, s>>>(a);
  else if (a.Dh <= 96) attn_seq_pp_kernel<PAGED, 6><<<grid, 512, 0, s>>>(a);
  else attn_seq_pp_kernel<PAGED, 8><<<grid, 512, 0, s>>>(a);
  return qie_last_error();
}

}  // namespace

int qie_launch_seq_pp(const SeqArgs& a, bool paged, hipStream_t s) {
  const int64_t rb = (int64_t)a.T * a.G / kPPRows + a.B;  // at least the row blocks of any lengths
  const int64_t grid = rb * (a.ct ? a.maxch : 1) * a.Hk;
  if (grid > INT32_MAX) return QIE_ERR_UNSUPPORTED;
  return paged ? launch<true>(a, (unsigned)grid, s) : launch<false>(a, (unsigned)grid, s);
}
