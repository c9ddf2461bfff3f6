// Rotary positions with several axes (time, height, width) on the heads of token rows, and the
// same rotation with the write of k and v into a paged cache.
//
// Pair i of a head turns by a_i = 2 pi frac(pos[axis[i]] * turns[i]), turns[i] full turns for each
// step of its axis (theta^(-i/n) / 2 pi). The product and its fraction are 64-bit: at position 1e5
// a 32-bit angle would be off by 2^-24 * 1e5 = 6e-3 rad, three quarters of a bf16 step; what is left
// after the fraction, |frac| <= 1/2, goes on in 32 bits. The rotation is fp32 with one rounding:
//   (x, y) -> (x cos a - y sin a, y cos a + x sin a),
// x and y half a rotary width apart (half) or neighbours (interleaved).
//
// Bound by HBM: every head is read and written once, the angles of a token are shared by all its
// heads. A work-group computes the cos / sin of its tokens once into LDS, then its threads walk the
// (token, head) items, V pairs each as 16-byte accesses. Measured (device, median): 16816 rows of 48 heads of
// 128 77 us into other memory, 5.4 TB/s, 61 in place, 6.7; the append of 4099 rows of 28 + 2 x 4 heads 14.1 us, 5.4 TB/s;
// up to some hundred rows the launch (16 rows 3.5 us, 300 rows of 32 heads 3.4, 784 of 32 80-wide heads 4.2).
#include <algorithm>

#include "qie_common.h"

namespace {

struct RopeArgs {
  const bf16_t* x;  // first rotated head of row 0
  int64_t ldx;
  bf16_t* out;  // where the rotated heads go (x itself: in place)
  int64_t ldo;
  int T, nh, hs, Dh;  // rows, rotated heads, head stride, head width
  const int* pos;     // [axes][T], row stride ldp
  int64_t ldp;
  int axes;
  const double* turns;  // [pairs]
  const int* axis;      // [pairs]
  int pairs, tb;        // rotary width / 2; tokens of a work-group
  // append: the first H of the nh = H + Hk heads are q; k and v go to the pages
  int H, Hk;
  bf16_t *kp, *vp;  // [pages][Hk][P][Dh]
  int64_t ps, hsp, ss;
  const int64_t* slots;
  int64_t nslots;
  int pshift;
};

template <int N>
struct Vec;
template <>
struct Vec<8> { typedef u32x4_t t; };
template <>
struct Vec<4> { typedef u32x2_t t; };
template <>
struct Vec<2> { typedef uint32_t t; };
template <>
struct Vec<1> { typedef bf16_t t; };

// N consecutive bf16 as one access (two 16-byte ones for N = 16)
template <int N>
__device__ __forceinline__ void load_n(const bf16_t* p, bf16_t* v) {
  constexpr int M = N > 8 ? 8 : N;
#pragma unroll
  for (int i = 0; i < N / M; ++i) {
    const typename Vec<M>::t w = *(const typename Vec<M>::t*)(p + i * M);
    __builtin_memcpy(v + i * M, &w, sizeof(w));
  }
}
template <int N>
__device__ __forceinline__ void store_n(bf16_t* p, const bf16_t* v) {
  constexpr int M = N > 8 ? 8 : N;
#pragma unroll
  for (int i = 0; i < N / M; ++i) {
    typename Vec<M>::t w;
    __builtin_memcpy(&w, v + i * M, sizeof(w));
    *(typename Vec<M>::t*)(p + i * M) = w;
  }
}

constexpr int kRopeTB = 4;       // most tokens of a work-group
constexpr int kRopePairs = 128;  // most pairs (head_dim <= 256)

template <int V, bool INTER, bool APPEND>
__global__ void __launch_bounds__(256) rope_axes_kernel(RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[2][kRopeTB * kRopePairs];  // cos, sin [token][pair]
  const int t0 = blockIdx.x * a.tb, nt = min(a.tb, a.T - t0);
  const int tid = threadIdx.x;
  for (int i = tid; i < nt * a.pairs; i += 256) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    const int ax = min(max(a.axis[p], 0), a.axes - 1);
    const double r = (double)a.pos[(int64_t)ax * a.ldp + t0 + t] * a.turns[p];
    float s, c;
    sincospif(2.0f * (float)(r - __builtin_rint(r)), &s, &c);
    cs[0][i] = c;
    cs[1][i] = s;
  }
  __syncthreads();
  // a thread keeps its V pairs and walks the (token, head) items
  const int upr = a.pairs / V, groups = 256 / upr;
  const int grp = tid / upr, p0 = (tid - grp * upr) * V;
  if (grp < groups)
    for (int i = grp; i < nt * a.nh; i += groups) {
      const int t = i / a.nh, h = i - t * a.nh;
      const bf16_t* src = a.x + (int64_t)(t0 + t) * a.ldx + (int64_t)h * a.hs;
      bf16_t* dst = a.out + (int64_t)(t0 + t) * a.ldo + (int64_t)h * a.hs;
      if constexpr (APPEND)
        if (h >= a.H) {
          const int64_t slot = a.slots[t0 + t];
          if (slot < 0 || slot >= a.nslots) continue;
          dst = a.kp + (slot >> a.pshift) * a.ps + (h - a.H) * a.hsp + (slot & ((1 << a.pshift) - 1)) * a.ss;
        }
      bf16_t v[2 * V];
      if constexpr (INTER) {
        load_n<2 * V>(src + 2 * p0, v);
      } else {
        load_n<V>(src + p0, v);
        load_n<V>(src + a.pairs + p0, v + V);
      }
      const float* ct = cs[0] + t * a.pairs + p0;
      const float* st = cs[1] + t * a.pairs + p0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int ix = INTER ? 2 * j : j, iy = INTER ? 2 * j + 1 : j + V;
        const float x = bf2f(v[ix]), y = bf2f(v[iy]), c = ct[j], s = st[j];
        v[ix] = f2bf(__builtin_fmaf(x, c, -(y * s)));
        v[iy] = f2bf(__builtin_fmaf(y, c, x * s));
      }
      if constexpr (INTER) {
        store_n<2 * V>(dst + 2 * p0, v);
      } else {
        store_n<V>(dst + p0, v);
        store_n<V>(dst + a.pairs + p0, v + V);
      }
    }
  // columns past the rotary width pass through where the heads go elsewhere
  const int rest = a.Dh - 2 * a.pairs;
  if (rest > 0)
    for (int i = tid; i < nt * a.nh * rest; i += 256) {
      const int th = i / rest, d = 2 * a.pairs + (i - th * rest), t = th / a.nh, h = th - t * a.nh;
      const bf16_t* src = a.x + (int64_t)(t0 + t) * a.ldx + (int64_t)h * a.hs + d;
      bf16_t* dst = a.out + (int64_t)(t0 + t) * a.ldo + (int64_t)h * a.hs + d;
      if constexpr (APPEND)
        if (h >= a.H) {
          const int64_t slot = a.slots[t0 + t];
          if (slot < 0 || slot >= a.nslots) continue;
          dst = a.kp + (slot >> a.pshift) * a.ps + (h - a.H) * a.hsp + (slot & ((1 << a.pshift) - 1)) * a.ss + d;
        }
      if (src != dst) *dst = *src;
    }
  if constexpr (APPEND) {  // v rows, unrotated: head_dim % 8 == 0, 16-byte chunks
    const int nch = a.Dh >> 3;
    for (int i = tid; i < nt * a.Hk * nch; i += 256) {
      const int th = i / nch, c = i - th * nch, t = th / a.Hk, h = th - t * a.Hk;
      const int64_t slot = a.slots[t0 + t];
      if (slot < 0 || slot >= a.nslots) continue;
      *(u32x4_t*)(a.vp + (slot >> a.pshift) * a.ps + h * a.hsp + (slot & ((1 << a.pshift) - 1)) * a.ss + c * 8) =
          *(const u32x4_t*)(a.x + (int64_t)(t0 + t) * a.ldx + (int64_t)(a.nh + h) * a.hs + c * 8);
    }
  }
}

// Tokens of a work-group: with fewer than 2048 rows one, so that the rows spread over the chip (300 rows of 32
// heads: 3.5 us, 4.3 with four); else as many as give its threads two items each, for the cos and sin of a
// token are made by the same threads (in place, 16384 rows of 8 heads: 11.0 us with four, 16.0 with one; 4096 of 32: 9.3
// with two, 10.3 with one; 16816 of 48: 61.3 with one, 63.4 with four).
int rope_tokens(const RopeArgs& a, int V) {
  if (a.T < 2048) return 1;
  return (int)std::min<int64_t>(kRopeTB, std::max<int64_t>(1, 2 * 256 / ((int64_t)a.nh * (a.pairs / V))));
}

template <bool APPEND>
int launch_rope(RopeArgs& a, bool inter, hipStream_t s) {
  // V pairs of a thread as 16-byte accesses need rows, heads and halves on 16 bytes; 8-byte ones and single
  // elements take the others (4096 rows of 32 heads in place: 9.3, 11.1 and 20.0 us)
  const uint64_t al = (uint64_t)a.x | (uint64_t)a.out | (uint64_t)(2 * (a.ldx | a.ldo | a.hs)) |
                      (uint64_t)(inter ? 0 : 2 * a.pairs);
#define ROPE_LAUNCH(V)                                                             \
  do {                                                                             \
    a.tb = rope_tokens(a, V);                                                      \
    const unsigned grid = (unsigned)((a.T + a.tb - 1) / a.tb);                     \
    if (inter) rope_axes_kernel<V, true, APPEND><<<grid, 256, 0, s>>>(a);          \
    else rope_axes_kernel<V, false, APPEND><<<grid, 256, 0, s>>>(a);               \
  } while (0)
  if (al % 16 == 0 && a.pairs % 8 == 0) ROPE_LAUNCH(8);
  else if (al % 16 == 0 && inter && a.pairs % 4 == 0) ROPE_LAUNCH(4);
  else if (al % 8 == 0 && a.pairs % 4 == 0 && !inter) ROPE_LAUNCH(4);
  else ROPE_LAUNCH(1);
#undef ROPE_LAUNCH
  return qie_last_error();
}

bool rope_common_ok(const void* x, const void* out, int rows, int head_dim, const int* positions, int64_t ldp,
                    int axes, const double* turns, const int* axis, int pairs) {
  return x && out && positions && turns && axis && rows >= 0 && head_dim > 0 && pairs > 0 && 2 * pairs <= head_dim &&
         pairs <= kRopePairs && axes > 0 && (ldp >= rows || ldp == 0) && (uintptr_t)x % 4 == 0 && (uintptr_t)out % 4 == 0 &&
         (uintptr_t)turns % 8 == 0;
}

}  // namespace

extern "C" int qie_rope_axes_bf16(const void* x, int64_t ldx, void* out, int64_t ldo, int rows, int heads,
                                  int head_dim, int head_stride, const int* positions, int64_t ldp, int axes,
                                  const double* turns, const int* axis, int pairs, int interleaved,
                                  qie_stream_t stream) {
  QIE_CHECK_ARG(rope_common_ok(x, out, rows, head_dim, positions, ldp, axes, turns, axis, pairs));
  QIE_CHECK_ARG(heads > 0 && head_stride >= head_dim && head_stride % 2 == 0 && ldx % 2 == 0 && ldo % 2 == 0);
  const int64_t width = (int64_t)(heads - 1) * head_stride + head_dim;
  QIE_CHECK_ARG(ldx >= width && ldo >= width && width <= INT32_MAX / kRopeTB);
  if (rows == 0) return QIE_OK;
  RopeArgs a{};
  a.x = (const bf16_t*)x;
  a.ldx = ldx;
  a.out = (bf16_t*)out;
  a.ldo = ldo;
  a.T = rows;
  a.nh = heads;
  a.hs = head_stride;
  a.Dh = head_dim;
  a.pos = positions;
  a.ldp = ldp;
  a.axes = axes;
  a.turns = turns;
  a.axis = axis;
  a.pairs = pairs;
  return launch_rope<false>(a, interleaved != 0, (hipStream_t)stream);
}

extern "C" int qie_rope_append_bf16(const void* qkv, int64_t ldx, void* q_out, int64_t ldo, int rows, int heads,
                                    int kv_heads, int head_dim, const int* positions, int64_t ldp, int axes,
                                    const double* turns, const int* axis, int pairs, int interleaved, void* k_pages,
                                    void* v_pages, int num_pages, int page_size, int64_t page_stride,
                                    int64_t page_head_stride, int64_t slot_stride, const int64_t* slots,
                                    qie_stream_t stream) {
  QIE_CHECK_ARG(rope_common_ok(qkv, q_out, rows, head_dim, positions, ldp, axes, turns, axis, pairs));
  QIE_CHECK_ARG(heads > 0 && kv_heads > 0 && head_dim % 8 == 0 && k_pages && v_pages && slots);
  QIE_CHECK_ARG(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0);
  const int64_t width = (int64_t)(heads + 2 * kv_heads) * head_dim;
  QIE_CHECK_ARG(ldx >= width && ldo >= (int64_t)heads * head_dim && width <= INT32_MAX / kRopeTB);
  QIE_CHECK_ARG(ldx % 8 == 0 && ldo % 8 == 0);
  QIE_CHECK_ARG(num_pages > 0 && page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0);
  QIE_CHECK_ARG(page_stride >= 0 && page_head_stride >= 0 && slot_stride >= head_dim &&
                (page_stride | page_head_stride | slot_stride) % 8 == 0);
  if (rows == 0) return QIE_OK;
  RopeArgs a{};
  a.x = (const bf16_t*)qkv;
  a.ldx = ldx;
  a.out = (bf16_t*)q_out;
  a.ldo = ldo;
  a.T = rows;
  a.nh = heads + kv_heads;
  a.hs = head_dim;
  a.Dh = head_dim;
  a.pos = positions;
  a.ldp = ldp;
  a.axes = axes;
  a.turns = turns;
  a.axis = axis;
  a.pairs = pairs;
  a.H = heads;
  a.Hk = kv_heads;
  a.kp = (bf16_t*)k_pages;
  a.vp = (bf16_t*)v_pages;
  a.ps = page_stride;
  a.hsp = page_head_stride;
  a.ss = slot_stride;
  a.slots = slots;
  a.nslots = (int64_t)num_pages * page_size;
  a.pshift = __builtin_ctz(page_size);
  return launch_rope<true>(a, interleaved != 0, (hipStream_t)stream);
}
