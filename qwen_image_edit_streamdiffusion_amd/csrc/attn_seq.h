// Shared pieces of the attention over sequences (attn_seq.hip: 64-row blocks, joins and dispatch;
// attn_seq_few.hip: 16 and 32; attn_seq_pp.hip: 256): arguments, where a work-group's item lies, tile loads,
// and what keeps infinities and NaN of masked keys away from the rows that do not see them.
#pragma once
#include "qie_common.h"

struct SeqArgs {
  const bf16_t* q;
  int64_t ldq, hsq;
  const bf16_t *k, *v;  // packed rows, or pages
  int64_t ldk, hsk;     // row (slot) and head strides
  bf16_t* out;
  int64_t ldo, hso;
  const int* cu;  // [B + 1] token offsets (nullptr: one token each)
  int B, T, H, Hk, G, Dh;
  int causal;
  float c;    // scale * log2(e)
  float low;  // "no key yet": below every score whose logit 32 bits hold, finite, so that exp2((-inf - low) c) is 0, not NaN
  // paged
  const int* table;
  int64_t ldt, ps;
  const int* kv_lens;
  int width, pages, pshift;
  // keys in chunks of ct tiles, fp32 partials (ct = 0: whole rows); rows of a block
  int ct, maxch, bm;
  int shares;  // 256-row blocks: work-groups that share each kv head's keys (0: a work-group a block)
  float* ws;  // chunks: O [T * H][maxch][Dh], then (m, l) [T * H][maxch][2]; shares: attn_seq_pp.hip
};

namespace {

constexpr int kKB = 64;      // keys of a tile, here the unit in which chunks are counted
constexpr int kRowB = 256;   // LDS row: 128 elements, narrower heads leave zeros
constexpr int kTile = kKB * kRowB;
constexpr float kRescale = 8.0f;   // lazy rescale threshold, log2 units

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ i32x4_t seq_rsrc(const bf16_t* base, int bytes) {
  const uint64_t p = (uint64_t)base;
  return i32x4_t{uni((int)(uint32_t)p), uni((int)(uint32_t)(p >> 32)), uni(bytes), 0x00020000};
}
// 1 KiB (4 LDS rows) straight from memory: lane i's 16 bytes go to dst + 16 i, zeros out of range
__device__ __forceinline__ void seq_dma(const i32x4_t& r, const char QIE_LDS* dst, uint32_t voff) {
  const int lds = uni((int)(uint32_t)(uintptr_t)dst);
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %1, 0 offen lds"
      :
      : "v"(voff), "s"(r), "s"(lds)
      : "memory", "m0");
}

// where item `idx` lies: sequence b, its first token, tokens n, keys kv, row block blk, key chunk ch
struct Item {
  int b, start, n, kv, blk, ch, nch;
};

template <bool PAGED>
__device__ __forceinline__ void seq_span(const SeqArgs& a, int b, int& start, int& n, int& kv) {
  int e;
  if (a.cu) {
    start = min(max(a.cu[b], 0), a.T);
    e = min(max(a.cu[b + 1], start), a.T);
  } else {
    start = min(b, a.T);
    e = min(b + 1, a.T);
  }
  n = e - start;
  kv = PAGED ? min(max(a.kv_lens[b], 0), a.width << a.pshift) : n;
}

// inclusive sum over the lanes: within rows of 16, then a row's last lane to the next row, then 31 to 32 ..
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// The idx-th (row block, key chunk) over all sequences: a wave-wide scan of the sequences' counts.
template <bool PAGED, int BM>
__device__ __forceinline__ bool find_item(const SeqArgs& a, int idx, Item& it) {
  const int lane = threadIdx.x & 63;
  if (!a.cu && !a.ct && a.G <= BM) {  // one token each, whole: item b is sequence b
    if (idx >= a.B) return false;
    it.b = idx;
    seq_span<PAGED>(a, idx, it.start, it.n, it.kv);
    it.blk = it.ch = 0;
    it.nch = 1;
    return it.n > 0;
  }
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int start = 0, n = 0, kv = 0, cnt = 0;
    if (b0 + lane < a.B) {
      seq_span<PAGED>(a, b0 + lane, start, n, kv);
      cnt = (n * a.G + BM - 1) / BM;
      if (a.ct) cnt *= max(1, (kv + a.ct * kKB - 1) / (a.ct * kKB));
    }
    const int pre = wave_scan(cnt);
    const unsigned long long hit = __ballot(pre > idx);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      it.b = b0 + l;
      it.start = __builtin_amdgcn_readlane(start, l);
      it.n = __builtin_amdgcn_readlane(n, l);
      it.kv = __builtin_amdgcn_readlane(kv, l);
      const int j = idx - __builtin_amdgcn_readlane(pre - cnt, l);
      if (j < 0 || j >= __builtin_amdgcn_readlane(cnt, l)) return false;  // offsets that overlap: sums past 32 bits
      it.nch = a.ct ? max(1, (it.kv + a.ct * kKB - 1) / (a.ct * kKB)) : 1;
      const int nblk = (it.n * a.G + BM - 1) / BM;
      it.ch = j / nblk;               // neighbours read the same keys
      it.blk = nblk - 1 - j % nblk;  // the longest rows of a causal sequence first
      return true;
    }
    idx -= __builtin_amdgcn_readlane(pre, 63);
  }
  return false;
}

// max / sum over the four lanes that hold a row (lanes l, l ^ 16, l ^ 32, l ^ 48) without LDS. The
// instruction itself: fmaxf first quiets the operands that came as integers, two more instructions a step
__device__ __forceinline__ float max_of(uint32_t x, uint32_t y) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
  return r;
}
__device__ __forceinline__ float quad_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = max_of(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_of(b[0], b[1]);
}
__device__ __forceinline__ float quad_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// After a row's maximum has moved: is some row's largest logit so far from 0 that fma(score, c, -(maximum c)), where
// one product is rounded and the other is not, is off by more than 2^-12 (half a unit of 4096)? At 1e10 it would be
// hundreds where it should be 0. All later tiles of such a wave come here and subtract the maximum from the scores
// themselves (mscale 0: not a second time). Costs 0.2 % of the mean call, 5 % of the worst (7 x 45 new tokens over 400).
constexpr float kFar = 4096.f;
__device__ __forceinline__ bool seq_far(const SeqArgs& a, float m_run, float& above, float& mscale) {
  const bool far = __any(fabsf(m_run * a.c) > kFar && m_run > a.low);
  above = far ? -INFINITY : kRescale;
  mscale = far ? 0.f : a.c;
  return far;
}

// Infinities and NaN among bf16 values: the largest magnitude so far, as integers, one per half
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
struct Magnitude {
  u16x2_t m = {0, 0};
  __device__ __forceinline__ void add(const bf16x8_t x) {
    const u32x4_t w = __builtin_bit_cast(u32x4_t, x);
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w.x & 0x7fff7fffu));
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w.y & 0x7fff7fffu));
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w.z & 0x7fff7fffu));
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w.w & 0x7fff7fffu));
  }
  __device__ __forceinline__ bool nonfinite() const { return m.x >= 0x7f80 || m.y >= 0x7f80; }
};
// the finite values of a fragment, 0 for the others
__device__ __forceinline__ bf16x8_t finite(bf16x8_t x) {
  const u32x4_t w = __builtin_bit_cast(u32x4_t, x);
  uint32_t o[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((o[i] & 0x7f80u) == 0x7f80u) o[i] &= 0xffff0000u;
    if ((o[i] & 0x7f800000u) == 0x7f800000u) o[i] &= 0xffffu;
  }
  return __builtin_bit_cast(bf16x8_t, u32x4_t{o[0], o[1], o[2], o[3]});
}
// an infinity or NaN of a value that the row sees (low or high half of a pair), else 0
__device__ __forceinline__ float special(uint32_t w, int high, bool see) {
  const float f = high ? hi_f(w) : lo_f(w);
  return see && (__float_as_uint(f) & 0x7f800000u) == 0x7f800000u ? f : 0.f;
}

}  // namespace

// attn_seq_pp.hip: blocks of kPPRows rows
constexpr int kPPRows = 256;
int qie_launch_seq_pp(const SeqArgs& a, bool paged, hipStream_t s);
// attn_seq_few.hip: blocks of a.bm = 16 or 32 rows, keys shared by 4 or 8 waves
int qie_launch_seq_few(const SeqArgs& a, bool paged, int waves, hipStream_t s);
