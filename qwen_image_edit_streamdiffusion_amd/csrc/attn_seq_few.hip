// Attention over sequences for few rows (single tokens, short chunks of new tokens): bound by the
// latency of a chain of loads where the cache is short, by HBM where it is long. One work-group =
// 16 MT rows (tokens x the G query heads of one kv head) of one sequence; its NW waves share the
// keys: wave w takes the 32-key tiles w, w + NW, ... of the item, each in a 16-KiB LDS image of its
// own, with no barrier until the end. K of the next tile is asked for as soon as this tile's scores
// are made, V as soon as its product is, so a wave always has 8 KiB on the way and a work-group
// 8 NW .. 16 NW KiB. At the end the waves' (max, sum, O) meet in LDS.
//
// Products as in attn_seq.hip (S^T = K Q^T and O^T += V^T P^T on mfma 16x16x32). Measured (device,
// median), 28 heads over 4: 48 single tokens over 900 .. 32768 keys 284 us, 5.6 TB/s, and 5.4 for the join; 16 over 70
// .. 600 7.6 us, 41 new tokens over 309 6.9 (latency: launch, length and table, two or three rounds of tiles, merge).
#include "attn_seq.h"

namespace {

constexpr int kFK = 32;                 // keys of a tile
constexpr int kFTile = kFK * kRowB;     // 8 KiB: K, then V

// Two waves a SIMD are what the LDS allows; said here, it keeps all registers of the four-wave form directly addressable
// (80 tokens over 20 keys 14.7 us, 16.2 where products went through accumulation registers).
template <bool PAGED, int NK, int MT, int NW>  // NK 32-wide steps of the head: head_dim <= 32 NK
__global__ void __launch_bounds__(64 * NW, 2) attn_seq_few_kernel(SeqArgs a) {
  constexpr int ND = 2 * NK;
  constexpr int BM = 16 * MT;
  __shared__ __attribute__((aligned(16))) char smem_raw[NW * 2 * kFTile];
  __shared__ __attribute__((aligned(8))) float ml[NW][BM][2];
  char QIE_LDS* smem = (char QIE_LDS*)smem_raw;

  const int hk = blockIdx.x % a.Hk;
  Item it;
  if (!find_item<PAGED, BM>(a, blockIdx.x / a.Hk, it)) return;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int g = lane >> 4, ql = lane & 15;
  const int rows = it.n * a.G, row0 = it.blk * BM;
  const int t0 = a.ct ? it.ch * a.ct * 2 : 0;

  // ---- tiles: two 16-row halves (a page holds 16 tokens at least), each four 1-KiB pieces
  const uint32_t ldb = (uint32_t)(a.ldk * 2);
  const int head_bytes = a.Dh * 2;
  char QIE_LDS* kt = smem + wave * 2 * kFTile;
  char QIE_LDS* vt = kt + kFTile;
  uint32_t ko[4], vo[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int row = 4 * p + g, ck = ql ^ row, cv = ql ^ ((row & 7) << 1);
    ko[p] = ck * 8 < a.Dh ? row * ldb + ck * 16 : 0x80000000u;
    vo[p] = cv * 8 < a.Dh ? row * ldb + cv * 16 : 0x80000000u;
  }
  const int* table = PAGED ? a.table + (int64_t)it.b * a.ldt : nullptr;
  int tb = t0 + wave, pg[2] = {0, 0};  // lane i: the pages of tile tb + i NW's halves (-1: outside the pool)
  auto pages = [&](int from) {
    tb = from;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t page = ((int64_t)(from + lane * NW) * kFK + 16 * h) >> a.pshift;
      int id = -1;
      if (page < a.width) id = table[page];
      pg[h] = id >= 0 && id < a.pages ? id : -1;
    }
  };
  // table entries and q are asked for before anything looks at the sequence's length, which arrives with them
  if constexpr (PAGED) pages(tb);
  bf16x8_t qf[MT][NK];
  int toks[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = min(row0 + 16 * mt + ql, rows - 1), head = hk * a.G + r % a.G;
    toks[mt] = r / a.G;
    const bf16_t* qr = a.q + (int64_t)(it.start + toks[mt]) * a.ldq + (int64_t)head * a.hsq;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      qf[mt][ks] = bf16x8_t{};
      if (32 * ks + 8 * g < a.Dh) qf[mt][ks] = *(const bf16x8_t*)(qr + 32 * ks + 8 * g);
    }
  }
  const int off = it.kv - it.n;
  const int last = (min(rows, row0 + BM) - 1) / a.G;
  const int most = a.causal ? min(it.kv, max(off + last + 1, 0)) : it.kv;
  const int ntot = (most + kKB - 1) / kKB;  // in the 64-key units that chunks are counted in
  if (it.ch > 0 && it.ch * a.ct >= ntot) return;  // a causal block that ends before this chunk
  const bool whole = !a.ct || ntot <= a.ct;
  const int t1 = min((most + kFK - 1) / kFK, a.ct ? t0 + 2 * a.ct : INT32_MAX);
  auto dma = [&](const bf16_t* base, char QIE_LDS* dst, const uint32_t (&voff)[4], int t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = t * kFK + 16 * h, nrow = min(16, it.kv - key);
      bool ok = nrow > 0;
      int64_t at;
      if constexpr (PAGED) {
        const int id = __builtin_amdgcn_readlane(pg[h], (t - tb) / NW);
        ok = ok && id >= 0;
        at = (int64_t)(ok ? id : 0) * a.ps + (int64_t)(key & ((1 << a.pshift) - 1)) * a.ldk;
      } else {
        at = ok ? (int64_t)(it.start + key) * a.ldk : 0;
      }
      const i32x4_t rs = seq_rsrc(base + at + (int64_t)hk * a.hsk, ok ? (nrow - 1) * (int)ldb + head_bytes : 0);
#pragma unroll
      for (int p = 0; p < 4; ++p) seq_dma(rs, dst + h * 4096 + p * 1024, voff[p]);
    }
  };
  int t = t0 + wave;
  if (t < t1) {
    dma(a.k, kt, ko, t);
    dma(a.v, vt, vo, t);
  }
  int lim[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) lim[mt] = a.causal ? min(it.kv, max(off + toks[mt] + 1, 0)) : it.kv;
  const int lim0 = uni(lim[0]);
  f32x4_t o[MT][ND];
  float m_run[MT], l_run[MT];
  float above[MT], mscale[MT];  // seq_far
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m_run[mt] = a.low;
    above[mt] = kRescale;
    mscale[mt] = a.c;
    l_run[mt] = 0.f;
#pragma unroll
    for (int db = 0; db < ND; ++db) o[mt][db] = f32x4_t{};
  }

  if (t < t1) __builtin_amdgcn_s_waitcnt(0);  // q as well: from here on the counter is the tiles'
  for (; t < t1; t += NW) {
    const bool more = t + NW < t1;
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // K(t); V(t) may be on its way
    f32x4_t s[MT][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) s[mt][kb] = f32x4_t{};
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        const bf16x8_t A = *(const bf16x8_t QIE_LDS*)(kt + (kb * 16 + ql) * kRowB + (((4 * ks + g) ^ ql) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, qf[mt][ks], s[mt][kb], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K's image is read: the next one may come
    if (more) {
      if constexpr (PAGED)
        if (t + NW - tb >= 64 * NW) {
          pages(t + NW);
          __builtin_amdgcn_s_waitcnt(0);
        }
      dma(a.k, kt, ko, t + NW);
    }
    const int kv0 = t * kFK;
    const bool masked = kv0 + kFK > lim0;
    bf16x8_t pf[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (masked) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (kv0 + (i >> 2) * 16 + 4 * g + (i & 3) >= lim[mt]) s[mt][i >> 2][i & 3] = -INFINITY;
      }
      float mx = s[mt][0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[mt][i >> 2][i & 3]);
      mx = quad_max(mx);
      if (__any((mx - m_run[mt]) * a.c > above[mt])) {
        const float m_new = fmaxf(m_run[mt], mx);
        const float alpha = __builtin_amdgcn_exp2f((m_run[mt] - m_new) * a.c);
        m_run[mt] = m_new;
        l_run[mt] *= alpha;
#pragma unroll
        for (int db = 0; db < ND; ++db) o[mt][db] *= alpha;
        if (__builtin_expect(seq_far(a, m_run[mt], above[mt], mscale[mt]), 0))
#pragma unroll
          for (int i = 0; i < 8; ++i) s[mt][i >> 2][i & 3] -= m_run[mt];
      }
      const float mc = m_run[mt] * mscale[mt];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][i >> 2][i & 3], a.c, -mc));
        l_run[mt] += p;
        pf[mt][i] = (__bf16)p;
      }
    }
    if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // V(t); K of the next tile may be on its way
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // V^T fragment: lane's d = 16 db + ql, keys 4 g + 0..3 and 16 further
    auto vfrag = [&](int db) -> bf16x8_t {
      const int row = 4 * g + (ql >> 2), ch = (2 * db + ((ql & 3) >> 1)) ^ ((row & 7) << 1);
      const char QIE_LDS* p0 = vt + row * kRowB + (ch << 4) + 8 * (ql & 1);
      const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t QIE_LDS*)p0);
      const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t QIE_LDS*)(p0 + 16 * kRowB));
      return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    Magnitude mag;  // 0 * inf and 0 * NaN: a masked key's V must not reach the rows that do not see it
    if (masked) {
#pragma unroll
      for (int db = 0; db < ND; ++db) mag.add(vfrag(db));
      asm volatile("" ::: "memory");
    }
    if (__builtin_expect(__any(mag.nonfinite()), 0)) {
#pragma unroll
      for (int db = 0; db < ND; ++db) {
        const bf16x8_t A = finite(vfrag(db));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, pf[mt], o[mt][db], 0, 0, 0);
      }
#pragma unroll 1
      for (int j = 0; j < kFK; ++j) {
        const char QIE_LDS* vr = vt + j * kRowB + 8 * (g & 1);
#pragma unroll
        for (int db = 0; db < ND; ++db) {
          const u32x2_t w = *(const u32x2_t QIE_LDS*)(vr + (((2 * db + (g >> 1)) ^ ((j & 7) << 1)) << 4));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[mt][db][i] += special(i < 2 ? w.x : w.y, i & 1, kv0 + j < lim[mt]);
        }
      }
    } else {
#pragma unroll
      for (int db = 0; db < ND; ++db) {
        const bf16x8_t A = vfrag(db);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, pf[mt], o[mt][db], 0, 0, 0);
      }
    }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      dma(a.v, vt, vo, t + NW);
    }
  }

  // ---- the waves' parts meet: fp32 rows in each wave's own image, 16-byte chunks swizzled by the row
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float l = quad_sum(l_run[mt]);
#pragma unroll
    for (int db = 0; db < ND; ++db)
      *(f32x4_t QIE_LDS*)(kt + (16 * mt + ql) * 512 + (((4 * db + g) ^ ql) << 4)) = o[mt][db];
    if (g == 0) {
      ml[wave][16 * mt + ql][0] = m_run[mt];
      ml[wave][16 * mt + ql][1] = l;
    }
  }
  __syncthreads();
  const int nc = a.Dh >> 2;  // chunks of four elements
  for (int u = threadIdx.x; u < BM * nc; u += 64 * NW) {
    const int row = u / nc, ch = u - row * nc, r = row0 + row;
    if (r >= rows) break;
    f32x2_t mw[NW];
    f32x4_t v[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      mw[w] = *(const f32x2_t QIE_LDS*)&ml[w][row][0];
      v[w] = *(const f32x4_t QIE_LDS*)(smem + w * 2 * kFTile + row * 512 + ((ch ^ (row & 15)) << 4));
    }
    float M = a.low;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, mw[w][0]);
    float L = 0.f;
    f32x4_t O = f32x4_t{};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f((mw[w][0] - M) * a.c);  // a wave that saw no key left zeros
      L = __builtin_fmaf(f, mw[w][1], L);
#pragma unroll
      for (int i = 0; i < 4; ++i) O[i] = __builtin_fmaf(f, v[w][i], O[i]);
    }
    const int tok = r / a.G, head = hk * a.G + r % a.G;
    if (whole) {
      const float inv = L == 0.f ? 0.f : 1.0f / L;
      *(u32x2_t*)(a.out + (int64_t)(it.start + tok) * a.ldo + (int64_t)head * a.hso + 4 * ch) =
          u32x2_t{pack2(O[0] * inv, O[1] * inv), pack2(O[2] * inv, O[3] * inv)};
    } else {
      const int64_t pi = ((int64_t)(it.start + tok) * a.H + head) * a.maxch + it.ch;
      *(f32x4_t*)(a.ws + pi * a.Dh + 4 * ch) = O;
      if (ch == 0) *(f32x2_t*)(a.ws + (int64_t)a.T * a.H * a.maxch * a.Dh + pi * 2) = f32x2_t{M, L};
    }
  }
}

template <bool PAGED, int MT, int NW>
int launch(const SeqArgs& a, unsigned grid, hipStream_t s) {
  if (a.Dh <= 64) attn_seq_few_kernel<PAGED, 2, MT, NW><<<grid, 64 * NW, 0, s>>>(a);
  else if (a.Dh <= 96) attn_seq_few_kernel<PAGED, 3, MT, NW><<<grid, 64 * NW, 0, s>>>(a);
  else attn_seq_few_kernel<PAGED, 4, MT, NW><<<grid, 64 * NW, 0, s>>>(a);
  return qie_last_error();
}

template <bool PAGED>
int launch_few(const SeqArgs& a, int waves, hipStream_t s) {
  const int64_t rb = (int64_t)a.T * a.G / a.bm + a.B;  // at least the row blocks of any lengths
  const int64_t grid = rb * a.maxch * a.Hk;
  if (grid > INT32_MAX) return QIE_ERR_UNSUPPORTED;
  if (a.bm == 16) return waves == 8 ? launch<PAGED, 1, 8>(a, (unsigned)grid, s) : launch<PAGED, 1, 4>(a, (unsigned)grid, s);
  if constexpr (PAGED) return launch<true, 2, 8>(a, (unsigned)grid, s);
  return QIE_ERR_UNSUPPORTED;
}

}  // namespace

int qie_launch_seq_few(const SeqArgs& a, bool paged, int waves, hipStream_t s) {
  return paged ? launch_few<true>(a, waves, s) : launch_few<false>(a, waves, s);
}
