// bounded.hip -- a cache of fixed size (mi_op_bounded_*, include/mi355_ops.h): append, attention of one new token that also says what weight
// every key received, the same weights for the queries of a prompt, eviction of the least weighted keys.
//
// The slot that a key lies in and its position in the sequence are two things here: after an eviction they differ.  Softmax does not ask for
// the order of keys (they are cached rotated), so a cache may hold them in any order, and an eviction moves the kept keys behind the new end
// into the holes in front of it and nothing else.
#include <algorithm>

#include "attn_prefill_body.h"

namespace mi {

namespace {

using prefill::f32x4;
using prefill::mfma16;
using prefill::pack2_split;
using prefill::u32x2;
using prefill::u32x4;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -3.402823466e38f;      // where a maximum starts: finite, so that its distance to -inf (a masked score) is no NaN
constexpr int MAX_SPLITS = 64;          // slices of a row's keys
constexpr int MAX_GROUP = 128;          // query heads per KV head

// exp(scale * (s - m)) of products s and m <= s's maximum, sc = scale * log2 e.  The difference first: at its maximum a score of any size weighs one (scale * s - scale * m in
// one fused operation leaves the rounding of scale * m, 2^5 where a score is 2^30).
__device__ __forceinline__ float weight_of(float s, float m, float sc) { return __builtin_amdgcn_exp2f((s - m) * sc); }
__device__ __forceinline__ float weight_of(float s, float m, float sc, float up) { return __builtin_amdgcn_exp2f(fmaf(s - m, sc, up)); }      // times 2^up

// The same for a sum whose maximum is m, of sums whose largest maximum is M: never quite zero, so that what is infinite in it stays infinite.
__device__ __forceinline__ float share_of(float m, float M, float sc) { return fmaxf(weight_of(m, M, sc), 1.401298464e-45f); }

__device__ __forceinline__ int held_keys(const BoundedCache& c, int r) { return min(max(c.len[r], 0), c.cap); }

// Places of 16 keys that begin at a multiple of 16: one block of a paged cache (blocks are powers of two from 16 on).  The index of the first
// key's row of D elements; -1 where the table names no block of the arena (its keys take no part).
__device__ __forceinline__ int64_t row_of_16(const BoundedCache& c, int r, int h, int key) {
  if (c.btab == nullptr) return ((int64_t)r * c.Hkv + h) * c.cap + key;
  const int blk = c.btab[(size_t)r * c.bt_stride + (key >> c.bs_shift)];
  if ((unsigned)blk >= (unsigned)c.n_blocks) return -1;
  return (((int64_t)blk * c.Hkv + h) << c.bs_shift) + (key & ((1 << c.bs_shift) - 1));
}

// Across a wave in the vector unit (data-parallel primitives: a shift inside a row of 16, the last lane of a row to the next ones); a shuffle goes through
// LDS, 120 cycles a step.  The last lane holds the whole.
template <typename F>
__device__ __forceinline__ int wave_scan(int v, int none, F&& f) {
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false));      // row_shr:1
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));      // row_bcast:15 into rows 1 and 3
  return f(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));   // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ int wave_scan_sum(int v) { return wave_scan(v, 0, [](int a, int b) { return a + b; }); }

// raw bits of NB bytes (2, or a multiple of 4)
template <int NB>
struct Raw { uint32_t w[(NB + 3) / 4]; };
template <int NB>
__device__ __forceinline__ Raw<NB> load_bits(const void* p) {
  Raw<NB> o;
  if constexpr (NB % 16 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 16; ++i) {
      const u32x4 v = ((const u32x4*)p)[i];
      o.w[4 * i] = v.x; o.w[4 * i + 1] = v.y; o.w[4 * i + 2] = v.z; o.w[4 * i + 3] = v.w;
    }
  } else if constexpr (NB % 8 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 8; ++i) {
      const u32x2 v = ((const u32x2*)p)[i];
      o.w[2 * i] = v.x; o.w[2 * i + 1] = v.y;
    }
  } else if constexpr (NB % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 4; ++i) o.w[i] = ((const uint32_t*)p)[i];
  } else {
    o.w[0] = *(const uint16_t*)p;
  }
  return o;
}

// ---- append ---------------------------------------------------------------------------------------------------------------------------
// One lane takes 8 + 8 elements of a head, i .. i + 8 and i + D / 2 .. i + D / 2 + 8 (the two halves of a rotation's pairs), a power of two of
// lanes a head.  All in 32 bits, rounded once, to what is stored.
// STEP (few tokens a row): a workgroup per row, which moves the row's length and next position itself.  Otherwise the tasks of all tokens lie
// side by side and a second launch moves them (its atomics would come to one address from 1536 workgroups).
// Bound by memory: 8 x 1024 float32 tokens of 48 heads of 128, 407 MB, 74 us (5.5 TB/s; a copy of 4 GiB: 4.65 read and written) + 5 for the second launch; a step by its launch and one round
// trip: 2.4 us for one row, 4.2 for 32.

template <typename T>
struct alignas(16) Vec8 { T v[8]; };

// (us, one launch / two: 1 token a row 2.9 / -, 4 tokens of 1 row 4.0 / 4.8, of 256 rows 6.3 / 8.3; 8 tokens 6.1 / 4.8, 6.9 / 5.8 for 64 rows)
constexpr int STEP_TASKS = 2048;

template <typename T, bool STEP>
__global__ __launch_bounds__(STEP ? 1024 : 256) void append_kernel(BoundedCache c, BoundedTokens t, int lane_bits) {
  const int nh = t.Hq + 2 * c.Hkv, D = c.D, D2 = D / 2, lanes = 1 << lane_bits;
  const int per_token = nh << lane_bits;
  const int64_t total = (STEP ? 1 : (int64_t)c.rows) * t.L * per_token;
  int n_step = 0, len_step = 0, next_step = 0;
  for (int64_t task = STEP ? threadIdx.x : (int64_t)blockIdx.x * 256 + threadIdx.x; task < total; task += STEP ? 1024 : total) {
    const int64_t token = (STEP ? (int64_t)blockIdx.x * t.L : 0) + (t.L == 1 && STEP ? 0 : STEP ? (uint32_t)task / (uint32_t)per_token : task / per_token);
    const int in_token = (int)(STEP ? (t.L == 1 ? task : (uint32_t)task % (uint32_t)per_token) : task % per_token);
    const int r = STEP ? blockIdx.x : (int)(token / t.L), i = (int)(token - (int64_t)r * t.L);
    const int head = in_token >> lane_bits, e0 = (in_token & (lanes - 1)) * 8;
    const int len = held_keys(c, r), next = c.next[r];
    const int n = t.count(c, r, len, next);
    const bool is_q = head < t.Hq, is_k = !is_q && head < t.Hq + c.Hkv;
    const bool has = e0 < D2;                    // (lanes beyond the head's size: D = 96, 192)
    Vec8<T> a{}, b{};
    T* dst = nullptr;
    if (i < n) {
      const T* src = (const T*)t.qkv + (int64_t)r * t.ld_row + (int64_t)i * t.ld_token + (int64_t)head * D + e0;
      if (has) { a = *(const Vec8<T>*)src; b = *(const Vec8<T>*)(src + D2); }
      if (is_q || is_k) {
        float x[8], y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { x[j] = (float)a.v[j]; y[j] = (float)b.v[j]; }
        const T* nw = (const T*)(is_q ? t.q_norm_w : t.k_norm_w);
        if (nw != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
          for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor(ss, o, 64);
          const float rs = 1.0f / sqrtf(ss / (float)D + t.eps);
          if (has) {
            const Vec8<T> wa = *(const Vec8<T>*)(nw + e0), wb = *(const Vec8<T>*)(nw + e0 + D2);
#pragma unroll
            for (int j = 0; j < 8; ++j) { x[j] *= rs * (float)wa.v[j]; y[j] *= rs * (float)wb.v[j]; }
          }
        }
        if (has) {
          const float* cp = t.cos_tab + (int64_t)(next + i) * D2 + e0;
          const float* sp = t.sin_tab + (int64_t)(next + i) * D2 + e0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            a.v[j] = (T)(x[j] * cp[j] - y[j] * sp[j]);
            b.v[j] = (T)(y[j] * cp[j] + x[j] * sp[j]);
          }
        }
      }
      if (!is_q) {
        const int kh = is_k ? head - t.Hq : head - t.Hq - c.Hkv, slot = len + i;
        const int64_t at = row_of_16(c, r, kh, slot & ~15);
        if (at >= 0) dst = (T*)(is_k ? c.k : c.v) + (at + (slot & 15)) * D + e0;
        if (is_k && e0 == 0) {
          const size_t m = ((size_t)r * c.Hkv + kh) * c.cap + slot;
          c.pos[m] = next + i;
          c.weight[m] = 0.f;
        }
      }
    }
    if (is_q) dst = (T*)t.q_out + (token * t.Hq + head) * D + e0;       // (zeros for tokens that are not taken)
    if (dst != nullptr && has) { *(Vec8<T>*)dst = a; *(Vec8<T>*)(dst + D2) = b; }
    n_step = n; len_step = len; next_step = next;
  }
  if constexpr (STEP) {
    __syncthreads();                             // every thread has read them
    if (threadIdx.x == 0) {
      c.len[blockIdx.x] = len_step + n_step;
      c.next[blockIdx.x] = next_step + n_step;
      if (t.taken != nullptr) t.taken[blockIdx.x] = n_step;
    }
  }
}

__global__ void advance_kernel(BoundedCache c, BoundedTokens t) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= c.rows) return;
  const int len = held_keys(c, r), next = c.next[r], n = t.count(c, r, len, next);
  c.len[r] = len + n;
  c.next[r] = next + n;
  if (t.taken != nullptr) t.taken[r] = n;
}

// ---- attend ---------------------------------------------------------------------------------------------------------------------------
// Everything is laid out so that nothing crosses lanes: S^T = K Q^T leaves in a lane the scores of one query head (its column, lane & 15) and of
// the keys that the same lane multiplies in O^T += V^T P^T, and every rescale is the lane's own.  16-bit: a tile is 32 keys, 16 x 16 x 32
// products; the slot k = 8 q + 4 t + i of the second product stands for key 16 t + 4 q + i (q = lane >> 4), which is where the first left
// it.  A lane loads E = D / 16 elements of 8 keys' values -- whole rows across 16 lanes -- and transposes its 8 x E block in registers
// (v_perm); column n of output tile j is element n E + j.  P goes in as two 16-bit terms, off by 2^-17 (bfloat16), 2^-22 (float16) of it at most.  float32: 16 x 16 x 4 products, no
// transposition.  The largest score so far is taken in when a new one exceeds it by 2^8 (float16: 2), not at every tile.
// float16 ends at 2^-24, and many keys far below the largest may be all there is where that one's value is small.  So P is 2^13 there, at most 2^15, where the score is the largest so far, and a tile whose
// largest is 2^11 below is raised until it is not, the sums with it: by a power of two, which rounds nothing, and down again behind it.  A weight is off by 2^-27 of the largest of its tile of 32 keys at most.
// What a key weighs needs the final maximum and sum of every head, so the products are kept (4 bytes a head and key, 3 % of 16-bit keys and values at 4 heads) and read by whoever has
// them: the workgroup itself where it is alone (`ALONE`), else the joining launch.  (Adding them from here, relative to the slice's maximum, would have needed the same second pass.)
// Bound by memory, once it runs: 4 x 32761 float16 keys, 32 / 8 heads of 128, 545 MB in 107 us (5.1 TB/s) + 9.6 to join; 32 rows of 0 to 2048 bf16 keys, 137 MB, 34 + 7.7 us, of which 4 + 5 are the
// launches' heads; 8 rows of 1025 float32 keys, 68 MB, 19.3 + 4.2: four of the 16 columns of a float32 product are heads, 4 us of matrix work that nothing hides in so short a call.

// P is 2^UP where the score is the largest, in the sums of weights and values alike.  Below one where values reach to the end of float32, whose sums then stay inside it: 2^16 of them at 2^8, the most that P
// goes beyond it.  (Values below 2^-102 lose bits for that.)
template <typename T>
constexpr float UP = std::is_same_v<T, f16> ? 13.f : -24.f;

// A row of D elements as an operand of the first product: 16-byte pieces, piece c of a lane from element (4 c + q) 16 bytes on.
template <typename T, int D>
struct Frag {
  static constexpr int PE = 16 / (int)sizeof(T), N = (D + 4 * PE - 1) / (4 * PE);
  u32x4 w[N];
  __device__ __forceinline__ void load(const T* row, int qd, bool ok = true) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int e = (4 * c + qd) * PE;
      if (D % (4 * PE) != 0) ok = ok && e < D;
      w[c] = ok ? *(const u32x4*)(row + e) : u32x4{0, 0, 0, 0};
    }
  }
};
template <typename T, int D>
__device__ __forceinline__ f32x4 dot16(const Frag<T, D>& a, const Frag<T, D>& b) {          // 16 rows of a by 16 rows of b
  f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < Frag<T, D>::N; ++c) {
    if constexpr (sizeof(T) == 2) {
      s = mfma16<T>(a.w[c], b.w[c], s);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w[c][e]), __uint_as_float(b.w[c][e]), s, 0, 0, 0);
    }
  }
  return s;
}

template <int E>
__device__ __forceinline__ u32x4 column(const Raw<E * 2> (&v)[8], int j) {         // element j of 8 rows
  uint32_t o[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    if constexpr (E == 1) o[p] = v[2 * p].w[0] | (v[2 * p + 1].w[0] << 16);
    else o[p] = __builtin_amdgcn_perm(v[2 * p + 1].w[j / 2], v[2 * p].w[j / 2], j & 1 ? 0x07060302u : 0x05040100u);
  }
  return u32x4{o[0], o[1], o[2], o[3]};
}

// An infinite value is infinite at any weight, but its product with a 16-bit weight's second term (zero, or of the other sign) is NaN, or with a weight that is zero in its type.  Where there are any
// (`INFINITE`: the sums of a first walk over the keys were not finite) they enter the products apart from the others, with one for a weight (zero for a score of -inf, which has none: bit 4 t + i of `some`).
// float32 has the one product: infinite, or NaN where the weight is zero in float32.
template <typename T>
__device__ __forceinline__ u32x4 infinite_ones(u32x4 a) {
  constexpr uint32_t INF = std::is_same_v<T, bf16> ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] &= ((a[i] & 0x7fffu) == INF ? 0xffffu : 0) | ((a[i] & 0x7fff0000u) == INF << 16 ? 0xffff0000u : 0);
  return a;
}

// O^T += V^T P^T for the keys of a tile: v[4 t + i] is this lane's E elements of key 16 t + 4 q + i, p[t][i] that key's weight
template <typename T, int E, bool INFINITE>
__device__ __forceinline__ void add_values(const Raw<E * 2> (&v)[8], const float (&p)[2][4], f32x4 (&o)[E], uint32_t some) {
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    pack2_split<T>(p[t][0], p[t][1], hi[2 * t], lo[2 * t]);
    pack2_split<T>(p[t][2], p[t][3], hi[2 * t + 1], lo[2 * t + 1]);
  }
  const u32x4 ph{hi[0], hi[1], hi[2], hi[3]}, pl{lo[0], lo[1], lo[2], lo[3]};
  u32x4 ones{0, 0, 0, 0};
  if constexpr (INFINITE) {
    constexpr uint32_t ONE = std::is_same_v<T, bf16> ? 0x3f80u : 0x3c00u;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i / 2] |= some >> i & 1 ? ONE << 16 * (i & 1) : 0;
  }
#pragma unroll
  for (int j = 0; j < E; ++j) {
    u32x4 a = column<E>(v, j);
    if constexpr (INFINITE) {
      const u32x4 b = infinite_ones<T>(a);
      a ^= b;
      o[j] = mfma16<T>(b, ones, o[j]);
      __builtin_amdgcn_sched_barrier(0);               // (one after the other: this rare way asks for no more registers than the other)
    }
    o[j] = mfma16<T>(a, ph, o[j]);
    o[j] = mfma16<T>(a, pl, o[j]);
  }
}
template <typename T, int E, int SUB>
__device__ __forceinline__ void add_values(const Raw<E * 4> (&v)[4 * SUB], const float (&p)[SUB][4], f32x4 (&o)[E]) {
#pragma unroll
  for (int t = 0; t < SUB; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[4 * t + i].w[j]), p[t][i], o[j], 0, 0, 0);
}

// Slices of a row's keys: at most `splits`, of a multiple of 128 keys each (one tile of 32 for each of four waves); up to 32 keys more are the last one's, not a slice of
// their own.
struct Slices { int keys, count; };
__device__ __forceinline__ Slices slices_of(int n, int splits) {
  Slices s;
  s.keys = ((max(n - 32, 1) + splits - 1) / splits + 127) & ~127;
  s.count = min(splits, (n + s.keys - 1) / s.keys);
  return s;
}

// Short caches: one workgroup takes all keys and query heads of a KV head (16 at a time) and keeps the scores in LDS.  Otherwise slices and a joining launch.
constexpr int ALONE_SCORES = 7168;                     // keys (in 32s) times heads: 28 KiB

// Workspace of a call in slices: scores [row][KV head][query head of the group][cap, in 32s] as products (no scale), then of every slice the largest score
// and the sum [row][KV head][slice][head][2], then its output [row][KV head][slice][head][D].
struct AttendWs {
  float* scores; float* stats; float* part; int ld;
};

// Waves a SIMD: as many as the first walk over the keys needs (the second, over infinite values, would ask for more registers where it is let).
template <typename T, int E, bool ALONE>
constexpr int attend_waves() {
  if (ALONE) return E > 8 ? 1 : 2;
  if (sizeof(T) == 4) return E <= 4 ? 4 : E <= 6 ? 3 : E <= 12 ? 2 : 1;
  return std::is_same_v<T, f16> ? (E == 1 ? 5 : E <= 4 ? 4 : E <= 8 ? 3 : E <= 12 ? 2 : 1) : (E == 1 ? 6 : E == 2 ? 5 : E <= 6 ? 4 : E <= 8 ? 3 : E <= 12 ? 2 : 1);
}

template <typename T, int E, bool ALONE>
__global__ __launch_bounds__(256, (attend_waves<T, E, ALONE>())) void attend_kernel(BoundedCache c, BoundedAttend a, AttendWs ws, int splits) {
  constexpr int D = 16 * E, NW = 4;
  constexpr int SUB = sizeof(T) == 4 && E > 8 ? 1 : 2, KT = 16 * SUB;      // (float32 heads of 192 and 256: registers for 16 keys)
  const int G = a.Hq / c.Hkv, split = blockIdx.x, kh = blockIdx.y % c.Hkv, r = blockIdx.y / c.Hkv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, qd = lane >> 4;
  const bool idle = a.counts != nullptr && a.counts[r] <= 0;
  const int n = idle ? 0 : held_keys(c, r);
  const Slices sl = ALONE ? Slices{n, 1} : slices_of(n, splits);
  if (!ALONE && split >= sl.count) return;              // (the joining launch knows which slices there are)
  const int s0 = split * sl.keys, s1 = split == sl.count - 1 ? n : s0 + sl.keys;

  __shared__ float sh_m[NW][16], sh_l[NW][16];
  __shared__ float sh_o[NW][16][D + 4];                 // (+ 4: the four quarters of a wave on different banks)
  __shared__ float all_m[ALONE ? MAX_GROUP : 1], all_r[ALONE ? MAX_GROUP : 1];
  __shared__ __align__(16) float all_s[ALONE ? ALONE_SCORES : 4];
  const float sc = a.scale * LOG2E;
  constexpr bool F16 = std::is_same_v<T, f16>;
  const float step = (F16 ? 1.f : 8.f) / sc;            // 2, 2^8
  for (int h0 = blockIdx.z * 16; h0 < G; h0 += 16 * gridDim.z) {
    const int heads = min(16, G - h0);
    T* out = (T*)a.out + ((size_t)r * a.Hq + kh * G + h0) * D;
    Frag<T, D> q, k[SUB];
    Raw<E * (int)sizeof(T)> v[4 * SUB];
    q.load((const T*)a.q + ((size_t)r * a.Hq + kh * G + h0 + ln) * D, qd, ln < heads);
    float m, l;
    f32x4 o[E];
    float* sc_out = ws.scores + ((size_t)(r * c.Hkv + kh) * G + h0 + ln) * ws.ld;      // (in slices)
    const int sh_at = (h0 + ln) * ws.ld;                                                // (alone)

    auto walk = [&](auto infinite) {                                     // true_type: 16-bit values that are infinite among them
      constexpr bool INFINITE = decltype(infinite)::value;
      m = LOWEST; l = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int base = s0 + wave * KT; base < s1; base += NW * KT) {
        bool there[SUB];
#pragma unroll
        for (int t = 0; t < SUB; ++t) {
          const int key = __builtin_amdgcn_readfirstlane(base + 16 * t);
          const int64_t at = key < s1 ? row_of_16(c, r, kh, key) : -1;
          there[t] = at >= 0;
          const int last = there[t] ? min(15, s1 - 1 - key) : 0;           // (a clamped address: its scores are masked, its values cleared)
          const T* kp = (const T*)c.k + (there[t] ? at : 0) * D;
          const T* vp = (const T*)c.v + (there[t] ? at : 0) * D;
          k[t].load(kp + (int64_t)min(ln, last) * D, qd);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * t + i] = load_bits<E * (int)sizeof(T)>(vp + (int64_t)min(4 * qd + i, last) * D + ln * E);
        }
        float p[SUB][4];
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < SUB; ++t) {
          f32x4 s = dot16(k[t], q);
          const int key = base + 16 * t + 4 * qd;
          if (base + KT > s1 || !there[t]) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (key + i >= s1 || !there[t]) {
                s[i] = -INFINITY;
#pragma unroll
                for (int w = 0; w < (int)(sizeof(v[0].w) / 4); ++w) v[4 * t + i].w[w] = 0;
              }
          }
          if (ln < heads && key < s1) {                                    // (`ld` reaches to the tile's end)
            if constexpr (ALONE) *(f32x4*)&all_s[sh_at + key] = s;
            else *(f32x4*)(sc_out + key) = s;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) { p[t][i] = s[i]; top = fmaxf(top, s[i]); }
        }
        if (__any(top > m + step)) {
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float now = fmaxf(m, top), f = INFINITE ? share_of(m, now, sc) : weight_of(m, now, sc);
          m = now; l *= f;
#pragma unroll
          for (int j = 0; j < E; ++j) o[j] *= f;
        }
        float up = UP<T>, down = 1.f;
        bool raised = false;
        if constexpr (F16) {
          raised = __any(top < m - 11.f / sc);
          if (raised) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float by = fminf(fmaxf(floorf((m - top) * sc), 0.f), 60.f);      // (sums are below 2^61)
            up += by;
            down = ldexpf(1.f, -(int)by);
#pragma unroll
            for (int j = 0; j < E; ++j) o[j] *= ldexpf(1.f, (int)by);
          }
        }
        uint32_t some = 0;
        if constexpr (INFINITE) {
#pragma unroll
          for (int i = 0; i < 4 * SUB; ++i) some |= p[i / 4][i % 4] > -INFINITY ? 1u << i : 0;
        }
#pragma unroll
        for (int t = 0; t < SUB; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[t][i] = weight_of(p[t][i], m, sc, up);
            l = F16 ? fmaf(p[t][i], down, l) : l + p[t][i];
          }
        if constexpr (sizeof(T) == 2) add_values<T, E, INFINITE>(v, p, o, some);
        else add_values<T, E, SUB>(v, p, o);
        if (raised) {
#pragma unroll
          for (int j = 0; j < E; ++j) o[j] *= down;
        }
      }
    };
    walk(std::false_type{});
    if constexpr (sizeof(T) == 2) {
      f32x4 odd{0.f, 0.f, 0.f, 0.f};                                     // (NaN once anything is not finite)
#pragma unroll
      for (int j = 0; j < E; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) odd[i] = fmaf(o[j][i], 0.f, odd[i]);
      if (__any((odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.f)) walk(std::true_type{});
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < 16) { sh_m[wave][ln] = m; sh_l[wave][ln] = l; }
    if (ln < heads) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < E; ++j) sh_o[wave][ln][(4 * qd + i) * E + j] = o[j][i];
    }
    __syncthreads();
    // the four waves' states
    auto join = [&](int h, float& M, float& L, float (&f)[NW]) {
      M = fmaxf(fmaxf(sh_m[0][h], sh_m[1][h]), fmaxf(sh_m[2][h], sh_m[3][h]));
      L = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) { f[w] = share_of(sh_m[w][h], M, sc); L = fmaf(sh_l[w][h], f[w], L); }
    };
    const size_t slice = ((size_t)(r * c.Hkv + kh) * splits + split) * G + h0;
    for (int e = threadIdx.x; e < heads * D; e += 256) {
      const int h = e / D, d = e % D;
      float M, L, f[NW], x = 0.f;
      join(h, M, L, f);
#pragma unroll
      for (int w = 0; w < NW; ++w) x = fmaf(sh_o[w][h][d], f[w], x);
      if constexpr (ALONE) {
        out[e] = (T)(L != 0.f ? x / L : 0.f);
      } else {
        ws.part[slice * D + e] = x;
        if (d == 0) { ws.stats[(slice + h) * 2] = M; ws.stats[(slice + h) * 2 + 1] = L; }
      }
    }
    if constexpr (ALONE) {
      if (threadIdx.x < heads) {
        float M, L, f[NW];
        join(threadIdx.x, M, L, f);
        all_m[h0 + threadIdx.x] = M;
        all_r[h0 + threadIdx.x] = L != 0.f ? 1.f / L : 0.f;
      }
      __syncthreads();
    }
  }
  if constexpr (ALONE) {                                // what every key received
    float* wp = c.weight + ((size_t)r * c.Hkv + kh) * c.cap;
    for (int key = threadIdx.x; key < n; key += 256) {
      const float w = wp[key];
      float x = 0.f;
      for (int h = 0; h < G; ++h) x = fmaf(weight_of(all_s[h * ws.ld + key], all_m[h], sc, UP<T>), all_r[h], x);
      wp[key] = w + x;
    }
  }
}

// The slices' results joined: the output, and the weights of JOIN_KEYS keys a workgroup, four a thread.  What depends on no result -- the scores of the first
// heads -- is on its way before the statistics are.
constexpr int JOIN_KEYS = 1024;

template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(BoundedCache c, BoundedAttend a, AttendWs ws, int splits) {
  constexpr int HB = 4;                                 // heads whose scores are loaded together
  const int G = a.Hq / c.Hkv, D = c.D, kh = blockIdx.y % c.Hkv, r = blockIdx.y / c.Hkv;
  const bool idle = a.counts != nullptr && a.counts[r] <= 0;
  const int n = idle ? 0 : held_keys(c, r);
  if (blockIdx.x > 0 && (int)blockIdx.x * JOIN_KEYS >= n) return;
  const int ns = slices_of(n, splits).count;            // (none where there are no keys)
  const int key = blockIdx.x * JOIN_KEYS + 4 * threadIdx.x;
  const float* sp = ws.scores + (size_t)(r * c.Hkv + kh) * G * ws.ld + min(key, max(0, ws.ld - 4));
  f32x4 s[HB];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int j = 0; j < HB; ++j) s[j] = *(const f32x4*)(sp + (size_t)min(h0 + j, G - 1) * ws.ld);
  };
  fetch(0);
  float* wp = c.weight + ((size_t)r * c.Hkv + kh) * c.cap;
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = wp[min(key + i, c.cap - 1)];
  // the output: its elements spread over the row's workgroups
  const int groups = max(1, (n + JOIN_KEYS - 1) / JOIN_KEYS);
  const float* st = ws.stats + (size_t)(r * c.Hkv + kh) * splits * G * 2;
  const float* pp = ws.part + (size_t)(r * c.Hkv + kh) * splits * G * D;
  float o[8], om[8];
  auto fetch_out = [&](int e, int i0) {
    const int ee = min(e, G * D - 1), h = ee / D;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const size_t i = (size_t)max(0, min(i0 + j, ns - 1)) * G;
      o[j] = pp[i * D + ee];
      om[j] = st[(i + h) * 2];
    }
  };
  const int e0 = blockIdx.x * 256 + threadIdx.x;
  fetch_out(e0, 0);
  const float sc = a.scale * LOG2E;
  __shared__ float sh_m[MAX_GROUP], sh_r[MAX_GROUP];
  for (int h = threadIdx.x >> 6; h < G; h += 4) {       // a wave per head, a lane per slice
    const int i = threadIdx.x & 63;
    const float2 v = *(const float2*)(st + ((size_t)max(0, min(i, ns - 1)) * G + h) * 2);
    const float M = __int_as_float(__builtin_amdgcn_readlane(wave_scan(__float_as_int(i < ns ? v.x : LOWEST), __float_as_int(LOWEST), [](int a, int b) {
      return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b))); }), 63));
    const float L = wave_sum(i < ns ? v.y * weight_of(v.x, M, sc) : 0.f);
    if (i == 0) { sh_m[h] = M; sh_r[h] = L != 0.f ? 1.f / L : 0.f; }
  }
  __syncthreads();
  if (key < n) {
    f32x4 x{0.f, 0.f, 0.f, 0.f};
    for (int h0 = 0; h0 < G; h0 += HB) {
      if (h0 > 0) fetch(h0);
#pragma unroll
      for (int j = 0; j < HB; ++j)
        if (h0 + j < G)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = fmaf(weight_of(s[j][i], sh_m[h0 + j], sc, UP<T>), sh_r[h0 + j], x[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (key + i < n) wp[key + i] = w[i] + x[i];
  }
  for (int e = e0; e < G * D; e += groups * 256) {
    const int h = e / D;
    float x = 0.f;
    for (int i0 = 0; i0 < ns; i0 += 8) {
      if (e != e0 || i0 > 0) fetch_out(e, i0);
#pragma unroll
      for (int j = 0; j < 8; ++j) x = i0 + j < ns ? fmaf(o[j], share_of(om[j], sh_m[h], sc), x) : x;
    }
    ((T*)a.out)[((size_t)r * a.Hq + kh * G) * D + e] = (T)(sh_r[h] != 0.f ? x * sh_r[h] : 0.f);      // (nothing to see: whatever the values are)
  }
}

// ---- weigh ----------------------------------------------------------------------------------------------------------------------------
// Queries of a row and KV head lie in one line, rho = query * G + head of the group, so that 128 of them see nearly the same keys.  Two passes
// over S^T = K Q^T: the largest score and the sum of every query (a lane keeps its own over the keys that it holds; four lanes join at the
// end), then the sum over the queries for every key.  The first keeps queries in registers and passes keys through LDS, the second the
// other way round.
// Bound by the matrix cores and the exponentials beside them, which hardly overlap: a block of 64 scores costs 16 cycles of the one and 15 to 20 of the other at D = 128.  4 prompts of 819 to 2048 bf16
// tokens, 32 / 8 heads: 64 + 72 + 5 us, 2 x 37 GFLOP, 560 TFLOP/s over both passes (a product of 8192 x 8192 x 8192: 1135; the clock under this load is 1.95 GHz).  2 prompts of 700 float32 tokens 58 + 5
// + 56 + 5 us, 70 TFLOP/s of 151.  The last 64 queries of 8001 paged keys 18 + 5 + 14 us, 10.5 GFLOP: units of four tiles each wait for their first keys.
// Workspace, rho of the queries that ask (`asking` a row at most): [row][KV head][rho][2]; with split keys [row][KV head][slice][rho][2] in front of the merge, and in the same place, with split
// queries, [slice][row][KV head][ld] sums.
struct WeighWs { float* stats; float* parts; float* sums; int ld; };

struct WeighRow {                                    // what the queries of a row are
  int n, first, queries, behind;                     // keys; first query that asks, their number; query i sees keys up to behind + i
};
__device__ __forceinline__ WeighRow weigh_row(const BoundedCache& c, const BoundedWeigh& a, int r) {
  WeighRow w;
  w.n = held_keys(c, r);
  const int cnt = a.counts != nullptr ? min(max(a.counts[r], 0), a.L) : a.L;
  w.first = a.last > 0 ? max(0, cnt - a.last) : 0;
  w.queries = cnt - w.first;
  w.behind = w.n - cnt;
  return w;
}

template <typename T, int D>
constexpr int tile_rows() { return D * (int)sizeof(T) <= 256 ? 64 : 32; }                  // rows of a tile in LDS: two tiles of 16 KiB

// 256 threads hold a tile of ROWS rows in registers on its way from memory to LDS.  Every row has an address (a load under a branch waits for all that
// are on their way); what is not there is masked where it is used.
template <typename T, int D, int ROWS>
struct Stage {
  static constexpr int PER = D * (int)sizeof(T) / 16, LD = D * (int)sizeof(T) + 16;        // pieces a row; bytes a row in LDS (16 more: rows on different banks)
  static constexpr int N = (ROWS * PER + 255) / 256;
  u32x4 w[N];
  static __device__ __forceinline__ int row(int s) { return min((int)(threadIdx.x + s * 256) / PER, ROWS - 1); }      // of this thread's piece s
  static __device__ __forceinline__ uint32_t piece(int s) { return (threadIdx.x + s * 256) % PER * 16; }              // its bytes in the row
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int s = 0; s < N; ++s) {
      const int p = threadIdx.x + s * 256;
      if (ROWS * PER % 256 == 0 || p < ROWS * PER) *(u32x4*)(lds + p / PER * LD + p % PER * 16) = w[s];
    }
  }
};

// keys that any of the `queries` queries from rho0 on sees
__device__ __forceinline__ int weigh_most(const WeighRow& w, int G, int rho0, int queries) {
  return w.behind + w.first + (min(w.queries * G, rho0 + queries) - 1) / G + 1;
}

// the compiler's order: N times a matrix instruction, then V vector instructions and X exponentials
template <int N, int V, int X>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
    __builtin_amdgcn_sched_group_barrier(0x400, X, 0);
  }
}

// What a workgroup of a pass takes: KV heads side by side (a head stays on one XCD where their number is a multiple of eight), then slices, then rows, then
// tiles, those with the most work first.  Rows change places from tile to tile: workgroups go round the shader engines in order, and where the n-th is always
// of the longest row, one engine gets all of those and the others wait behind it (4 prompts of up to 2048 tokens: 472 of 1024 places taken for the first 60 us of 88).
struct WeighPlace { int r, kh, slice, tile; };
__device__ __forceinline__ WeighPlace weigh_place(const BoundedCache& c, int slices) {
  const int x = blockIdx.x / c.Hkv, y = x / slices, tile = y / c.rows;
  return {(y + tile) % c.rows, (int)(blockIdx.x % c.Hkv), x % slices, tile};
}

// Queries of a workgroup of the first pass: U tiles of 16 a wave.  16 bits: two (four: 102 us instead of 88 for the pass over 4 prompts of up to 2048 tokens, two waves a SIMD; one: 106);
// float32, whose tiles cost eight times as much: one (2 prompts of 700 tokens, both passes: 123 us, with two 130).
template <typename T>
constexpr int weigh_queries() { return sizeof(T) == 4 ? 64 : 128; }

// ALONE: a workgroup holds all queries of a KV head (few of them, before few keys) and walks the keys twice, statistics first, then weights, summed over its columns: one launch, no
// workspace.
template <typename T, int E, bool ALONE>
__global__ __launch_bounds__(256, sizeof(T) == 2 && E <= 8 && !ALONE ? 3 : 2) void weigh_stats_kernel(BoundedCache c, BoundedWeigh a, WeighWs ws, int splits, int chunk) {
  constexpr int D = 16 * E, ROWS = tile_rows<T, D>(), QUERIES = weigh_queries<T>(), U = QUERIES / 64;
  using St = Stage<T, D, ROWS>;
  const int G = a.Hq / c.Hkv;
  const int qtiles = gridDim.x / (c.rows * c.Hkv * splits);
  const WeighPlace at = weigh_place(c, splits);
  const int r = at.r, kh = at.kh, split = at.slice;
  const WeighRow w = weigh_row(c, a, r);
  const int rho0 = (qtiles - 1 - at.tile) * QUERIES, rhos = w.queries * G;       // (the queries that see most keys first)
  if (rho0 >= rhos) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, qd = lane >> 4;
  __shared__ __align__(16) char tiles[2][ROWS * St::LD];
  __shared__ bool lost[2][ROWS / 16];
  __shared__ float sums[ALONE ? 2 : 1][4][ROWS];

  Frag<T, D> q[U];
  int sees[U];                                           // keys that the column's query sees
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int rho = rho0 + (wave * U + u) * 16 + ln;
    const int i = w.first + rho / G, g = rho % G;
    sees[u] = rho < rhos ? w.behind + i + 1 : 0;
    q[u].load((const T*)a.q + (((size_t)r * a.L + min(i, a.L - 1)) * a.Hq + kh * G + g) * D, qd, rho < rhos);
  }
  // the keys of this slice that any query of the workgroup sees, and how many of them all see
  const int most = weigh_most(w, G, rho0, QUERIES);
  const int all = rho0 + QUERIES <= rhos ? w.behind + w.first + rho0 / G + 1 : 0;
  const int s0 = split * chunk, s1 = min(most, s0 + chunk);
  if (s0 >= s1 && split > 0) return;                     // (the merge knows which slices there are)
  const float sc = a.scale * LOG2E;
  float m[U], l[U];
#pragma unroll
  for (int u = 0; u < U; ++u) { m[u] = LOWEST; l[u] = 0.f; }
  St st;
  // Not paged: a tile lies in one piece, behind one address.  Paged: the blocks of the tile after the next one are looked up in time.
  int block[St::N];
  bool gone[St::N];
  const int mask = (1 << c.bs_shift) - 1;
  const int32_t* table = c.btab != nullptr ? c.btab + (size_t)r * c.bt_stride : nullptr;
  const char* row0 = (const char*)c.k + ((int64_t)r * c.Hkv + kh) * c.cap * D * (int)sizeof(T);
  auto look = [&](int base) {
    if (table == nullptr) return;
#pragma unroll
    for (int s = 0; s < St::N; ++s) block[s] = table[min(base + St::row(s), s1 - 1) >> c.bs_shift];
  };
  auto fetch = [&](int base) {
    if (table == nullptr) {
      const char* from = row0 + (int64_t)base * D * (int)sizeof(T);
      const int left = s1 - base;
      if (left >= ROWS) {
#pragma unroll
        for (int s = 0; s < St::N; ++s) st.w[s] = *(const u32x4*)(from + (uint32_t)(St::row(s) * D * (int)sizeof(T) + St::piece(s)));
      } else {
#pragma unroll
        for (int s = 0; s < St::N; ++s) st.w[s] = *(const u32x4*)(from + (uint32_t)(min(St::row(s), left - 1) * D * (int)sizeof(T) + St::piece(s)));
      }
    } else {
#pragma unroll
      for (int s = 0; s < St::N; ++s) {
        gone[s] = (unsigned)block[s] >= (unsigned)c.n_blocks;
        const int64_t at = (((int64_t)(gone[s] ? 0 : block[s]) * c.Hkv + kh) << c.bs_shift) + (min(base + St::row(s), s1 - 1) & mask);
        st.w[s] = *(const u32x4*)((const char*)c.k + at * (D * (int)sizeof(T)) + St::piece(s));
      }
    }
  };
  auto put = [&](int buf) {                              // keys in a block that is none: marked, 16 at a time
    st.store(tiles[buf]);
    if (table != nullptr) {
#pragma unroll
      for (int s = 0; s < St::N; ++s)
        if ((threadIdx.x + s * 256) % (16 * St::PER) == 0) lost[buf][St::row(s) / 16] = gone[s];
    }
  };
  float inv[U];
  auto walk = [&](auto second) {
    if (s0 < s1) {
      look(s0);
      fetch(s0);
      look(s0 + ROWS);
      put(0);
    }
    __syncthreads();
    int cur = 0;
    for (int base = s0; base < s1; base += ROWS, cur ^= 1) {
      const bool more = base + ROWS < s1;
      if (more) {
        fetch(base + ROWS);
        look(base + 2 * ROWS);
      }
      const char* tile = tiles[cur];
      bool edge = base + ROWS > min(all, s1);
      if (table != nullptr) {
#pragma unroll
        for (int t = 0; t < ROWS / 16; ++t) edge = edge || lost[cur][t];
      }
      // 32 keys at a time; their products run while the exponentials of the 32 in front of them do
      auto keys = [&](auto masked) {
        f32x4 sv[2][2][U];
        auto products = [&](int t0, f32x4 (&o)[2][U]) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            Frag<T, D> k;
            k.load((const T*)(tile + ((t0 + t) * 16 + ln) * St::LD), qd);
#pragma unroll
            for (int u = 0; u < U; ++u) o[t][u] = dot16(k, q[u]);
          }
        };
        products(0, sv[0]);
#pragma unroll
        for (int t0 = 0; t0 < ROWS / 16; t0 += 2) {
          if (t0 + 2 < ROWS / 16) products(t0 + 2, sv[(t0 / 2 + 1) & 1]);
          f32x4 (&s)[2][U] = sv[(t0 / 2) & 1];
          if constexpr (decltype(masked)::value) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int key = base + (t0 + t) * 16 + 4 * qd;
              const bool there = table == nullptr || !lost[cur][t0 + t];
#pragma unroll
              for (int u = 0; u < U; ++u) {
                const int left = there ? min(sees[u], s1) - key : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (i >= left) s[t][u][i] = -INFINITY;
              }
            }
          }
          if constexpr (decltype(second)::value) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float x = 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u) x = fmaf(weight_of(s[t][u][i], m[u], sc), inv[u], x);
                x = row16_sum(x);
                if (ln == 0) sums[cur][wave][(t0 + t) * 16 + 4 * qd + i] = x;
              }
            continue;
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float top = s[0][u][0];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][u][i]);
            top = fmaxf(m[u], top);
            float x = l[u] * weight_of(m[u], top, sc), y = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x += weight_of(s[0][u][i], top, sc);
              y += weight_of(s[1][u][i], top, sc);
            }
            m[u] = top; l[u] = x + y;
          }
          if constexpr (sizeof(T) == 2 && !decltype(masked)::value) interleave<2 * U * Frag<T, D>::N, 3, 1>();
        }
      };
      if (edge) keys(std::true_type{});
      else keys(std::false_type{});
      const bool there = (int)threadIdx.x < ROWS && base + (int)threadIdx.x < s1 && (table == nullptr || !lost[cur][threadIdx.x / 16]);
      if (more) put(cur ^ 1);
      __syncthreads();
      if constexpr (decltype(second)::value) {
        if (there) {
          float* wp = c.weight + ((size_t)r * c.Hkv + kh) * c.cap + base + threadIdx.x;
          *wp += (sums[cur][0][threadIdx.x] + sums[cur][1][threadIdx.x]) + (sums[cur][2][threadIdx.x] + sums[cur][3][threadIdx.x]);
        }
      }
    }
  };
  walk(std::false_type{});
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
      const float mo = __shfl_xor(m[u], off, 64), lo = __shfl_xor(l[u], off, 64), M = fmaxf(m[u], mo);
      l[u] = l[u] * weight_of(m[u], M, sc) + lo * weight_of(mo, M, sc);
      m[u] = M;
    }
    if constexpr (ALONE) {
      inv[u] = l[u] != 0.f ? 1.f / l[u] : 0.f;
      continue;
    }
    const int rho = rho0 + (wave * U + u) * 16 + ln;
    if (qd == 0 && rho < rhos) {
      const size_t R = (size_t)a.asking() * G, rk = (size_t)r * c.Hkv + kh;
      if (splits == 1) {
        ws.stats[(rk * R + rho) * 2] = l[u] != 0.f ? m[u] : 0.f;
        ws.stats[(rk * R + rho) * 2 + 1] = l[u] != 0.f ? 1.f / l[u] : 0.f;
      } else {
        float* o = ws.parts + ((rk * splits + split) * R + rho) * 2;
        o[0] = m[u]; o[1] = l[u];
      }
    }
  }
  if constexpr (ALONE) walk(std::true_type{});
}

__global__ __launch_bounds__(256) void weigh_merge_kernel(BoundedCache c, BoundedWeigh a, WeighWs ws, int splits, int chunk, int queries) {
  const int G = a.Hq / c.Hkv, r = blockIdx.y / c.Hkv;
  const WeighRow w = weigh_row(c, a, r);
  const int rho = blockIdx.x * 256 + threadIdx.x;
  if (rho >= w.queries * G) return;
  const size_t R = (size_t)a.asking() * G, rk = blockIdx.y;
  const int have = max(1, (weigh_most(w, G, rho / queries * queries, queries) + chunk - 1) / chunk);       // slices with keys that the query's workgroups saw
  const float sc = a.scale * LOG2E;
  float M = LOWEST, L = 0.f;
  for (int i0 = 0; i0 < have; i0 += 8) {               // (eight loads on their way together)
    float2 p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = *(const float2*)(ws.parts + ((rk * splits + min(i0 + j, have - 1)) * R + rho) * 2);
    float top = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, p[j].x);
    L *= weight_of(M, top, sc);
    M = top;
#pragma unroll
    for (int j = 0; j < 8; ++j) L = i0 + j < have ? fmaf(p[j].y, weight_of(p[j].x, M, sc), L) : L;
  }
  ws.stats[(rk * R + rho) * 2] = L != 0.f ? M : 0.f;
  ws.stats[(rk * R + rho) * 2 + 1] = L != 0.f ? 1.f / L : 0.f;
}

// Tiles of the second pass: ROWS queries of one head, those of a head one after the other, from the first query on that sees the workgroup's first
// key.  A slice is `per` tiles; with more than one of them the sums of each go to the workspace and a third launch adds them in order.
struct WeighTiles { int i0, per_head, total; };
__device__ __forceinline__ WeighTiles weigh_tiles(const WeighRow& w, int G, int j0, int rows) {
  WeighTiles t;
  t.i0 = max(0, j0 - w.behind - w.first);
  t.per_head = (max(0, w.queries - t.i0) + rows - 1) / rows;
  t.total = t.per_head * G;
  return t;
}

template <typename T, int E, int KS>
__global__ __launch_bounds__(256, sizeof(T) == 2 && E <= 8 ? 3 : 2) void weigh_add_kernel(BoundedCache c, BoundedWeigh a, WeighWs ws, int per, int slices) {
  constexpr int D = 16 * E, ROWS = tile_rows<T, D>();
  using St = Stage<T, D, ROWS>;
  const int G = a.Hq / c.Hkv;
  const WeighPlace at = weigh_place(c, slices);
  const int r = at.r, kh = at.kh;
  const WeighRow w = weigh_row(c, a, r);
  const int j0 = at.tile * 64 * KS;
  if (j0 >= w.n) return;
  const WeighTiles wt = weigh_tiles(w, G, j0, ROWS);
  const int t0 = at.slice * per, t1 = min(wt.total, t0 + per);
  if (t0 >= t1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, qd = lane >> 4;
  __shared__ __align__(16) char tiles[2][ROWS * St::LD];
  __shared__ float2 stats[2][ROWS];

  const int my0 = j0 + wave * 16 * KS;
  Frag<T, D> k[KS];
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    const int key = my0 + 16 * t;
    const int64_t row = key < w.n ? row_of_16(c, r, kh, key) : -1;
    k[t].load((const T*)c.k + ((row < 0 ? 0 : row) + min(ln, max(0, w.n - 1 - key))) * D, qd, row >= 0);
  }
  const float sc = a.scale * LOG2E;
  const size_t rk = (size_t)r * c.Hkv + kh;
  const float* st_row = ws.stats + rk * a.asking() * G * 2;
  const T* q_row = (const T*)a.q + (((size_t)r * a.L + w.first) * a.Hq + kh * G) * D;
  const int64_t ld_q = (int64_t)a.Hq * D;
  float x[KS][4];
#pragma unroll
  for (int t = 0; t < KS; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[t][i] = 0.f;
  St st;
  float2 sv = make_float2(0.f, 0.f);
  uint32_t off[St::N];                                 // of this thread's pieces from a tile's first row
#pragma unroll
  for (int s = 0; s < St::N; ++s) off[s] = (uint32_t)(St::row(s) * ld_q * sizeof(T)) + St::piece(s);
  auto fetch = [&](int g, int first) {                 // queries first .. first + ROWS of head g; the last one again behind it, where it weighs nothing
    const int left = w.queries - first;
    const char* from = (const char*)(q_row + first * ld_q + g * D);
    const float* stat = st_row + ((size_t)first * G + g) * 2;
    if (left >= ROWS) {
#pragma unroll
      for (int s = 0; s < St::N; ++s) st.w[s] = *(const u32x4*)(from + off[s]);
      sv = *(const float2*)(stat + (threadIdx.x % ROWS) * G * 2);
    } else {
#pragma unroll
      for (int s = 0; s < St::N; ++s) st.w[s] = *(const u32x4*)(from + min((int64_t)St::row(s), (int64_t)left - 1) * ld_q * sizeof(T) + St::piece(s));
      sv = *(const float2*)(stat + min((int)threadIdx.x % ROWS, left - 1) * G * 2);
      if ((int)threadIdx.x >= left) sv = make_float2(INFINITY, 0.f);
    }
  };
  int g = t0 / wt.per_head, it = t0 % wt.per_head;
  fetch(g, wt.i0 + it * ROWS);
  st.store(tiles[0]);
  if (threadIdx.x < ROWS) stats[0][threadIdx.x] = sv;
  __syncthreads();
  int cur = 0;
  for (int tt = t0; tt < t1; ++tt, cur ^= 1) {
    const int first = wt.i0 + it * ROWS;
    if (++it == wt.per_head) { it = 0; ++g; }
    const bool more = tt + 1 < t1;
    if (more) fetch(g, wt.i0 + it * ROWS);
    const char* tile = tiles[cur];
    const int sees0 = w.behind + w.first + first + 1;    // keys that the tile's first query sees
    // the products of 16 queries run while the exponentials of the 16 in front of them do
    auto columns = [&](auto edge) {
      f32x4 sv2[2][KS];
      auto products = [&](int u, f32x4 (&o)[KS]) {
        Frag<T, D> q;
        q.load((const T*)(tile + (u * 16 + ln) * St::LD), qd);
#pragma unroll
        for (int t = 0; t < KS; ++t) o[t] = dot16(k[t], q);
      };
      products(0, sv2[0]);
#pragma unroll
      for (int u = 0; u < ROWS / 16; ++u) {
        if (u + 1 < ROWS / 16) products(u + 1, sv2[(u + 1) & 1]);
        const float2 ml = stats[cur][u * 16 + ln];
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float p = weight_of(sv2[u & 1][t][i], ml.x, sc);
            if (decltype(edge)::value && my0 + 16 * t + 4 * qd + i >= sees0 + u * 16 + ln) p = 0.f;
            x[t][i] = fmaf(p, ml.y, x[t][i]);
          }
        if constexpr (sizeof(T) == 2) interleave<KS * Frag<T, D>::N, 2, 1>();
      }
    };
    if (sees0 < my0 + 16 * KS) columns(std::true_type{});
    else columns(std::false_type{});
    if (more) {
      st.store(tiles[cur ^ 1]);
      if (threadIdx.x < ROWS) stats[cur ^ 1][threadIdx.x] = sv;
    }
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    const int key0 = my0 + 16 * t;
    const bool there = key0 < w.n && row_of_16(c, r, kh, key0) >= 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = row16_sum(x[t][i]);
      const int key = key0 + 4 * qd + i;
      if (ln != 0 || key >= w.n) continue;
      if (slices > 1) ws.sums[((size_t)at.slice * c.rows * c.Hkv + rk) * ws.ld + key] = there ? y : 0.f;
      else if (there) c.weight[rk * c.cap + key] += y;
    }
  }
}

__global__ __launch_bounds__(256) void weigh_sum_kernel(BoundedCache c, BoundedWeigh a, WeighWs ws, int per, int keys, int rows) {
  const int G = a.Hq / c.Hkv, r = blockIdx.y / c.Hkv, key = blockIdx.x * 256 + threadIdx.x;
  const WeighRow w = weigh_row(c, a, r);
  if (key >= w.n) return;
  const int slices = (weigh_tiles(w, G, key / keys * keys, rows).total + per - 1) / per;
  const float* p = ws.sums + (size_t)blockIdx.y * ws.ld + key;
  const size_t step = (size_t)c.rows * c.Hkv * ws.ld;
  float x = 0.f;
#pragma unroll 8
  for (int i = 0; i < slices; ++i) x += p[i * step];
  if (slices > 0) c.weight[(size_t)blockIdx.y * c.cap + key] += x;
}

// ---- evict ----------------------------------------------------------------------------------------------------------------------------
// A workgroup per row and KV head finds the budget-th largest of its keys' ranks (32-bit numbers in the order of the weights, protected keys
// above all): a histogram over the range that is left, 2048 bins, until a bin stays whole -- at most three, one or two where the weights differ.  A
// second launch moves keys and values: with the moves known it spreads over the chip.
// 64 rows and heads of 8192 keys down to 1024: 12.5 us (a chain of barriers on 64 CUs; the first histogram's range is wasted on the gap between zero and the least weight) + 15.7 us to move 59 MB (3.8 TB/s in rows of
// 256 bytes); 256 of 1025 down to 1024, in one launch: 8.4.
struct EvictWs { int32_t* counts; int2* moves; uint32_t* ranks; int most; };      // [row][KV head]; [row][KV head][most] (from, to); [row][KV head][cap]

// Where more keys are protected than the budget holds, they alone are ranked (`crowded`).  A slot in a block that is none has no key: in front of `budget` it stays as it is (no hole, as nothing can be
// written there), behind it it leaves.  Every other slot in front of `budget` holds a key, so there are always enough of them for what is left of the budget, and no move begins or ends in such a block.
constexpr uint32_t RANK_STAYS = 0xffffffffu, RANK_LEAVES = 0;
__device__ __forceinline__ uint32_t rank_of(float w, int pos, int first, int recent_from, bool crowded) {
  if ((pos < first || pos >= recent_from) != crowded) return crowded ? RANK_LEAVES : RANK_STAYS;
  if (w != w) w = -INFINITY;
  const uint32_t b = __float_as_uint(w + 0.f);                     // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// keys, values, positions and weights of `count` moves, by `threads` threads; no slot is both left and taken
__device__ __forceinline__ void move_rows(const BoundedCache& c, int r, int kh, int row_pieces, const int2* moves, int count, int thread, int threads) {
  const size_t rk = (size_t)r * c.Hkv + kh;
  float* w = c.weight + rk * c.cap;
  int32_t* q = c.pos + rk * c.cap;
  for (int e = thread; e < count; e += threads) {
    const int2 m = moves[e];
    w[m.y] = w[m.x];
    q[m.y] = q[m.x];
  }
  const int64_t total = (int64_t)count * row_pieces;
  for (int64_t e = thread; e < total; e += threads) {
    const int2 m = moves[e / row_pieces];
    const int p = (int)(e % row_pieces);
    const int64_t from = row_of_16(c, r, kh, m.x & ~15), to = row_of_16(c, r, kh, m.y & ~15);
    if (from < 0 || to < 0) continue;                              // (the selection has seen to that)
    const int64_t a = (from + (m.x & 15)) * row_pieces + p, b = (to + (m.y & 15)) * row_pieces + p;
    ((u32x4*)c.k)[b] = ((const u32x4*)c.k)[a];
    ((u32x4*)c.v)[b] = ((const u32x4*)c.v)[a];
  }
}

// exclusive sum of v over the workgroup's threads, the sum of all in total
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int& total, int* sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, incl = wave_scan_sum(v);
  if (lane == 63) sh[wave] = incl;
  __syncthreads();
  const int w = wave_scan_sum(lane < THREADS / 64 ? sh[lane] : 0);
  __syncthreads();
  total = __builtin_amdgcn_readlane(w, THREADS / 64 - 1);
  const int u = __builtin_amdgcn_readfirstlane(wave);
  return (u > 0 ? __builtin_amdgcn_readlane(w, u - 1) : 0) + incl - v;
}

// MOVE: the workgroup moves keys and values itself, from a list in LDS, and the row's last one sets its length (a ticket of the cache's, back at zero then; nothing
// waits for it).  For caches that can hold few keys beyond the budget: a step's eviction is one launch (32 rows of 8 heads, 1025 keys to 1024: 8.5 us, in two 6.5 + 3 and 3 us more of host time).
constexpr int MOVE_MOST = 64;
// slots whose ranks fit the LDS of a CU: 149 KiB
constexpr int ON_CHIP = 36864;      // (8 heads of 32768 keys down to 4096: 45 us; weights and positions read again at every sweep 70)
// IN_LDS: the ranks stay on chip, slot i at i + i / 32 (a thread's slots lie side by side, threads' on different banks); otherwise they lie in the workspace
template <bool IN_LDS, bool MOVE>
__global__ __launch_bounds__(1024) void evict_select_kernel(BoundedCache c, int budget, int keep_first, int keep_last, int row_pieces, EvictWs ws) {
  constexpr int THREADS = 1024, BINS = 2048, PER = BINS / THREADS, FEW = 4;       // (256 threads: 12.4 us for 8.8)
  const int r = blockIdx.y, kh = blockIdx.x, n = held_keys(c, r);
  const size_t rk = (size_t)r * c.Hkv + kh;
  auto leave = [&]() {                                             // (MOVE; in front of it every wave has read the length, or has one that stays as it is)
    if (threadIdx.x != 0 || atomicAdd(&c.tickets[r], 1) != c.Hkv - 1) return;
    c.len[r] = min(n, budget);
    __hip_atomic_store(&c.tickets[r], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  if (n <= budget) {
    if (MOVE) leave();
    else if (threadIdx.x == 0) ws.counts[rk] = 0;
    return;
  }
  float* wp = c.weight + rk * c.cap;
  int32_t* pp = c.pos + rk * c.cap;
  const int recent_from = (int)max((int64_t)c.next[r] - keep_last, (int64_t)INT32_MIN);
  extern __shared__ uint32_t lds_ranks[];
  uint32_t* ranks = IN_LDS ? lds_ranks : ws.ranks + rk * c.cap;
  __shared__ uint32_t hist[BINS];
  __shared__ int scan[16];
  __shared__ uint32_t sh_lo[16], sh_hi[16];
  __shared__ int sh_prot[16], sh_bin, sh_above, sh_in;
  bool crowded = false;
  auto rank = [&](int i) -> uint32_t& { return IN_LDS ? lds_ranks[i + (i >> 5)] : ranks[i]; };
  const int32_t* table = c.btab != nullptr ? c.btab + (size_t)r * c.bt_stride : nullptr;

  // ranks, their range, and how many keys stay whatever their weight
  uint32_t lo, hi;
  int prot;
  for (int turn = 0; turn < 2; ++turn) {
    lo = 0xffffffffu; hi = 0; prot = 0;
    for (int i0 = threadIdx.x; i0 < n; i0 += 8 * THREADS) {        // (the loads of eight slots on their way together)
      float w[8];
      int32_t p[8], block[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) { const int i = min(i0 + j * THREADS, n - 1); w[j] = wp[i]; p[j] = pp[i]; block[j] = table != nullptr ? table[i >> c.bs_shift] : 0; }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = i0 + j * THREADS;
        if (i >= n) continue;
        const bool lost = table != nullptr && (unsigned)block[j] >= (unsigned)c.n_blocks;
        const uint32_t k = lost ? (i < budget ? RANK_STAYS : RANK_LEAVES) : rank_of(w[j], p[j], keep_first, recent_from, crowded);
        rank(i) = k;
        if (k == RANK_STAYS) ++prot;
        else if (k != RANK_LEAVES) { lo = min(lo, k); hi = max(hi, k); }
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) hist[threadIdx.x + i * THREADS] = 0;
    lo = (uint32_t)wave_scan((int)lo, -1, [](int a, int b) { return (int)min((uint32_t)a, (uint32_t)b); });
    hi = (uint32_t)wave_scan((int)hi, 0, [](int a, int b) { return (int)max((uint32_t)a, (uint32_t)b); });
    prot = wave_scan_sum(prot);
    if ((threadIdx.x & 63) == 63) { sh_lo[threadIdx.x >> 6] = lo; sh_hi[threadIdx.x >> 6] = hi; sh_prot[threadIdx.x >> 6] = prot; }
    __syncthreads();
    lo = sh_lo[0]; hi = sh_hi[0]; prot = sh_prot[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) { lo = min(lo, sh_lo[w]); hi = max(hi, sh_hi[w]); prot += sh_prot[w]; }
    if (prot <= budget) break;
    crowded = true;
    __syncthreads();
  }
  // all ranks above `cut` stay, of those equal to it the `need` lowest slots
  uint32_t cut = RANK_STAYS - 1;
  int need = 0;
  bool found = false;
  if (n - budget <= FEW && !crowded) {                             // few leave: the least weighted alone (always, where it is one key a step; 9.8 -> 6.5 us of selection)
    int least = 0, all;
    for (int i = threadIdx.x; i < n; i += THREADS) least += rank(i) <= lo;         // (and the slots without a key)
    block_scan<THREADS>(least, all, scan);
    if (n - all <= budget) {
      cut = lo;
      need = budget - (n - all);
      found = true;
    }
  }
  if (prot < budget && !found) {
    need = budget - prot;
    for (;;) {                                                     // the range [lo, hi] holds the rank; it shrinks by a factor of 1024 at least
      const int shift = max(0, 21 - __clz(hi - lo | 1u));
      constexpr int BATCH = IN_LDS ? 4 : 16;
      for (int i0 = threadIdx.x; i0 < n; i0 += BATCH * THREADS) {
        uint32_t k[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) k[j] = rank(min(i0 + j * THREADS, n - 1));
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
          if (i0 + j * THREADS < n && k[j] >= lo && k[j] <= hi) atomicAdd(&hist[(k[j] - lo) >> shift], 1u);
      }
      __syncthreads();
      // bins from the highest down, PER a thread
      int h[PER], sum = 0, all;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int b = BINS - 1 - PER * (int)threadIdx.x - i;
        h[i] = (int)hist[b];
        hist[b] = 0;
        sum += h[i];
      }
      sum = block_scan<THREADS>(sum, all, scan);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (sum < need && sum + h[i] >= need) { sh_bin = BINS - 1 - PER * (int)threadIdx.x - i; sh_above = sum; sh_in = h[i]; }
        sum += h[i];
      }
      __syncthreads();
      need -= sh_above;
      lo += (uint32_t)sh_bin << shift;
      if (sh_in == need) {                                         // the whole bin stays
        cut = lo - 1;
        need = 0;
        break;
      }
      if (shift == 0) {
        cut = lo;
        break;
      }
      hi = min(hi, lo + ((1u << shift) - 1u));
    }
  }
  // in the order of slots, four a thread and turn: which stay, and the i-th hole in front of `budget` gets the i-th that stays behind it
  __shared__ int2 sh_moves[MOVE ? MOVE_MOST : 1];
  int2* moves = MOVE ? sh_moves : ws.moves + rk * ws.most;
  int equal0 = 0, holes0 = 0, movers0 = 0;
  uint32_t ahead[4];                                               // the next turn's
#pragma unroll
  for (int j = 0; j < 4; ++j) ahead[j] = rank(min(4 * (int)threadIdx.x + j, n - 1));
  for (int base = 0; base < n; base += 4 * THREADS) {
    const int i0 = base + 4 * threadIdx.x;
    uint32_t k[4];
    int equal = 0, all_equal = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k[j] = i0 + j < n ? ahead[j] : 0;
      if (i0 + j < n && k[j] == cut) ++equal;
    }
    if (base + 4 * THREADS < n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) ahead[j] = rank(min(i0 + 4 * THREADS + j, n - 1));
    }
    int at = equal0 + (need > 0 ? block_scan<THREADS>(equal, all_equal, scan) : 0), both = 0, all;
    bool stays[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      stays[j] = i0 + j < n && (k[j] > cut || (k[j] == cut && at < need));
      if (i0 + j < n && k[j] == cut) ++at;
      if (i0 + j < budget && !stays[j]) both += 1 << 16;         // (at most 4096 of either in a turn)
      if (i0 + j >= budget && stays[j]) both += 1;
    }
    both = block_scan<THREADS>(both, all, scan);
    int holes = holes0 + (both >> 16), movers = movers0 + (both & 0xffff);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + j < budget && !stays[j]) moves[holes++].y = i0 + j;
      if (i0 + j >= budget && stays[j]) moves[movers++].x = i0 + j;
    }
    equal0 += all_equal; holes0 += all >> 16; movers0 += all & 0xffff;
  }
  if constexpr (MOVE) {
    __syncthreads();
    move_rows(c, r, kh, row_pieces, sh_moves, movers0, threadIdx.x, THREADS);
    leave();
  } else {
    if (threadIdx.x == 0) ws.counts[rk] = movers0;
  }
}

__global__ __launch_bounds__(256) void evict_move_kernel(BoundedCache c, int budget, int row_pieces, EvictWs ws) {
  const int r = blockIdx.y / c.Hkv, kh = blockIdx.y % c.Hkv;
  if (blockIdx.x == 0 && kh == 0 && threadIdx.x == 0) c.len[r] = min(held_keys(c, r), budget);       // (nothing else of this launch reads it)
  move_rows(c, r, kh, row_pieces, ws.moves + (size_t)blockIdx.y * ws.most, ws.counts[blockIdx.y], blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------

template <typename F>
int by_type(int dtype, F&& f) {
  switch (dtype) {
    case MI_F32: return f(float{});
    case MI_BF16: return f(bf16{});
    case MI_F16: return f(f16{});
  }
  return fail(MI_ERR_INVALID, "bounded cache: dtype");
}
template <typename F>
int by_head(int D, F&& f) {                              // (mi_op_bounded_* have looked it over: bounded_head_dim)
  switch (D) {
    case 16: return f(std::integral_constant<int, 1>{});
    case 32: return f(std::integral_constant<int, 2>{});
    case 64: return f(std::integral_constant<int, 4>{});
    case 96: return f(std::integral_constant<int, 6>{});
    case 128: return f(std::integral_constant<int, 8>{});
    case 192: return f(std::integral_constant<int, 12>{});
    case 256: return f(std::integral_constant<int, 16>{});
  }
  return fail(MI_ERR_UNSUPPORTED, "bounded cache: head_dim");
}

// 321 keys of 8 KV heads: 8.7 us alone, in slices 10.8
bool attend_alone(const BoundedCache& c, int Hq) {
  const int G = Hq / c.Hkv;
  return c.cap <= 512 && c.cap * ((G + 15) / 16) <= 1024 && ((c.cap + 31) & ~31) * G <= ALONE_SCORES;
}
// Slices of a row's keys, of u times 128: so many workgroups that they fill two rounds of two a CU (rows are of unequal lengths; long caches, whose slices are, one round) and leave little of
// the last round empty.  (Two a CU is what float32 heads of 128 hold; 16-bit heads of 128 hold three, smaller ones more, and their slices were chosen by the times below, not by a count of their own.)  us, 1 / 2 / 3 units a slice: 32 rows of 520 float32 keys, 40 / 8 heads, 37.5 / 44.4 / 37.4; 8 of 2815 46.3 / 45.3 / 43.5; 8 of 1025 24.8 / 27.8 (21.4 without a slice for the last key); 4 of 32761 float16 keys in 16 /
// 32 / 64 slices 117 / 120 / 126; 32 of 0 to 2048 in 2 / 4 / 8 47.4 / 44.0 / 46.8.
int attend_splits(const BoundedCache& c, int Hq, int ncu) {
  const int64_t tiles = (int64_t)c.rows * c.Hkv * ((Hq / c.Hkv + 15) / 16), units = std::max(1, (c.cap - 32 + 127) / 128), slots = 2 * ncu;
  const int64_t rounds = c.cap >= 16384 ? 1 : 2, least = (units + MAX_SPLITS - 1) / MAX_SPLITS;
  const int64_t u0 = std::max(least, (tiles * units + slots * rounds / 2) / (slots * rounds)), from = u0 <= 4 ? least : std::max(least, u0 - 2), to = u0 <= 4 ? 2 * u0 + 2 : u0 + 2;
  int64_t best = 1, best_off = 0;
  double best_fill = 0;
  for (int64_t u = std::min(from, units); u <= std::min(to, units); ++u) {
    const int64_t s = (units + u - 1) / u, n = (tiles * s + slots - 1) / slots, off = std::abs(n - rounds);
    const double fill = (double)(tiles * s) / (double)(n * slots);
    if (fill > 1.05 * best_fill || (fill > 0.95 * best_fill && off <= best_off)) { best = s; best_off = off; best_fill = std::max(fill, best_fill); }
  }
  return (int)best;
}

// All queries of a KV head in one workgroup: where there are few of them, before few keys or in rows and heads enough to fill the chip.  us, alone / in units: 30 queries of 30 keys 7.3 /
// 12.3, 32 of 256 15.2 / 17.6, 32 of 400 23.3 / 17.3; float32 16 of 100 16.8 / 17.8, of 200 26.1 / 21.8; 64 rows of 8 heads, 32 queries, 400 keys 36 / 61, 4000 keys 294 / 407, float32 16 of 400 84 / 153;
// 256 rows and heads of 1000 keys 53 / 58; 200 of 300 keys, 3 queries, 18 / 52.
bool weigh_alone(const BoundedCache& c, const BoundedWeigh& a, int ncu) {
  const bool f32 = c.dtype == MI_F32;
  const int64_t L = a.asking();
  if (L * (a.Hq / c.Hkv) > (f32 ? weigh_queries<float>() : weigh_queries<bf16>())) return false;
  return c.cap <= (f32 ? 128 : 288) || 4 * c.rows * c.Hkv >= 3 * ncu;
}

// How a call is cut: units of nearly equal size, several times as many as the chip holds at once, so that its queues even them out.  First pass: 64 U queries by
// `chunk` keys; second: 64 KS keys by `per` tiles of queries.
struct WeighPlan { int splits, chunk, ks, per, slices; };
WeighPlan weigh_plan(const BoundedCache& c, const BoundedWeigh& a, int ncu) {
  WeighPlan p;
  const int G = a.Hq / c.Hkv, L = a.asking(), f32 = c.dtype == MI_F32, U = f32 ? 1 : 2;
  const int64_t pairs = (int64_t)c.rows * c.Hkv, groups = pairs * (((int64_t)L * G + 64 * U - 1) / (64 * U));
  const int64_t fit = std::max<int64_t>({(int64_t)c.cap * groups / ((f32 ? 16 : 8) * ncu), 256, (c.cap + MAX_SPLITS - 1) / MAX_SPLITS});
  p.chunk = (int)std::min<int64_t>((fit + 63) / 64 * 64, (c.cap + 63) / 64 * 64);
  p.splits = (c.cap + p.chunk - 1) / p.chunk;
  auto key_tiles = [&](int ks) { return pairs * ((c.cap + 64 * ks - 1) / (64 * ks)); };
  p.ks = !f32 && key_tiles(2) >= ncu ? 2 : 1;
  const int rows = c.D * (int)dtype_size(c.dtype) <= 256 ? 64 : 32;
  const int64_t tiles = (int64_t)G * ((L + rows - 1) / rows), least = f32 ? 4 : 8;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({MAX_SPLITS, 24 * ncu / key_tiles(p.ks), (tiles + least - 1) / least}));
  p.per = (int)((tiles + want - 1) / want);
  p.slices = (int)((tiles + p.per - 1) / p.per);
  return p;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

bool bounded_head_dim(int D) { return D == 16 || D == 32 || D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }
bool bounded_group(int G) { return G >= 1 && G <= MAX_GROUP; }

// (a launch takes fewer than 2^32 threads; one that fails would leave those behind it with what it has not written)
static int append_lane_bits(int D) {
  int bits = 0;
  while ((16 << bits) < D) ++bits;
  return bits;
}
bool bounded_append_fits(const BoundedCache& c, const BoundedTokens& t) {
  return (int64_t)c.rows * t.L <= (((int64_t)1 << 32) - 256) / ((t.Hq + 2 * c.Hkv) << append_lane_bits(c.D));
}
bool bounded_weigh_fits(const BoundedCache& c, const BoundedWeigh& a, int ncu) {
  if (weigh_alone(c, a, ncu)) return true;
  const WeighPlan p = weigh_plan(c, a, ncu);
  const int64_t Q = c.dtype == MI_F32 ? weigh_queries<float>() : weigh_queries<bf16>(), pairs = (int64_t)c.rows * c.Hkv, most = (1 << 24) - 1;
  return ((int64_t)a.asking() * (a.Hq / c.Hkv) + Q - 1) / Q * p.splits <= most / pairs && ((int64_t)c.cap + 64 * p.ks - 1) / (64 * p.ks) * p.slices <= most / pairs;
}

size_t bounded_attend_ws(const BoundedCache& c, int Hq, int ncu) {
  if (attend_alone(c, Hq)) return 0;
  const size_t splits = attend_splits(c, Hq, ncu), ld = ((size_t)c.cap + 31) & ~(size_t)31;
  return up256((size_t)c.rows * Hq * ld * 4) + up256((size_t)c.rows * Hq * splits * 8) + up256((size_t)c.rows * Hq * splits * c.D * 4);
}
size_t bounded_weigh_ws(const BoundedCache& c, const BoundedWeigh& a, int ncu) {
  if (weigh_alone(c, a, ncu)) return 0;
  const WeighPlan p = weigh_plan(c, a, ncu);
  const size_t one = up256((size_t)c.rows * a.Hq * a.asking() * 8), ld = ((size_t)c.cap + 3) & ~(size_t)3;
  return one + std::max(p.splits > 1 ? one * p.splits : 0, p.slices > 1 ? (size_t)p.slices * c.rows * c.Hkv * ld * 4 : 0);
}
size_t bounded_evict_ws(const BoundedCache& c, int budget) {
  const int most = std::min(budget, c.cap - budget);
  if (most <= 0) return 0;                               // (no row can hold more)
  const size_t pairs = (size_t)c.rows * c.Hkv;
  return (most > MOVE_MOST ? up256(pairs * 4) + up256(pairs * most * 8) : 0) + (c.cap > ON_CHIP ? pairs * c.cap * 4 : 0);
}

int launch_bounded_append(const BoundedCache& c, const BoundedTokens& t, hipStream_t st) {
  const int bits = append_lane_bits(c.D);
  return by_type(c.dtype, [&](auto z) {
    using T = decltype(z);
    if ((int64_t)t.L * (t.Hq + 2 * c.Hkv) << bits <= STEP_TASKS) {
      hipLaunchKernelGGL((append_kernel<T, true>), dim3(c.rows), dim3(1024), 0, st, c, t, bits);
    } else {
      const int64_t tasks = (int64_t)c.rows * t.L * (t.Hq + 2 * c.Hkv) << bits;
      hipLaunchKernelGGL((append_kernel<T, false>), dim3((unsigned)((tasks + 255) / 256)), dim3(256), 0, st, c, t, bits);
      hipLaunchKernelGGL(advance_kernel, dim3((c.rows + 63) / 64), dim3(64), 0, st, c, t);
    }
    MI_HIP(hipGetLastError());
    return MI_OK;
  });
}

int launch_bounded_attend(const BoundedCache& c, const BoundedAttend& a, void* ws, int ncu, hipStream_t st) {
  const int splits = attend_splits(c, a.Hq, ncu), G = a.Hq / c.Hkv;
  AttendWs w;
  w.ld = (c.cap + 31) & ~31;
  w.scores = (float*)ws;
  w.stats = (float*)((char*)ws + up256((size_t)c.rows * a.Hq * w.ld * 4));
  w.part = (float*)((char*)w.stats + up256((size_t)c.rows * a.Hq * splits * 8));
  return by_type(c.dtype, [&](auto z) {
    using T = decltype(z);
    return by_head(c.D, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (attend_alone(c, a.Hq)) {
        hipLaunchKernelGGL((attend_kernel<T, E, true>), dim3(1, c.rows * c.Hkv), dim3(256), 0, st, c, a, w, 1);
      } else {
        hipLaunchKernelGGL((attend_kernel<T, E, false>), dim3(splits, c.rows * c.Hkv, (G + 15) / 16), dim3(256), 0, st, c, a, w, splits);
        hipLaunchKernelGGL((attend_join_kernel<T>), dim3((c.cap + JOIN_KEYS - 1) / JOIN_KEYS, c.rows * c.Hkv), dim3(256), 0, st, c, a, w, splits);
      }
      MI_HIP(hipGetLastError());
      return MI_OK;
    });
  });
}

int launch_bounded_weigh(const BoundedCache& c, const BoundedWeigh& a, void* ws, int ncu, hipStream_t st) {
  const WeighPlan p = weigh_plan(c, a, ncu);
  const int G = a.Hq / c.Hkv, L = a.asking();
  float* more = (float*)((char*)ws + up256((size_t)c.rows * a.Hq * L * 8));
  const WeighWs w{(float*)ws, more, more, (c.cap + 3) & ~3};
  const unsigned rhos = (unsigned)L * G, pairs = c.rows * c.Hkv;
  return by_type(c.dtype, [&](auto z) {
    using T = decltype(z);
    return by_head(c.D, [&](auto e) {
      constexpr int E = decltype(e)::value;
      constexpr int Q = weigh_queries<T>(), KS = sizeof(T) == 4 ? 1 : 2;
      const dim3 queries((rhos + Q - 1) / Q * p.splits * pairs), keys((c.cap + 64 * p.ks - 1) / (64 * p.ks) * p.slices * pairs);
      if (weigh_alone(c, a, ncu)) {
        hipLaunchKernelGGL((weigh_stats_kernel<T, E, true>), dim3(pairs), dim3(256), 0, st, c, a, w, 1, c.cap);
        MI_HIP(hipGetLastError());
        return MI_OK;
      }
      hipLaunchKernelGGL((weigh_stats_kernel<T, E, false>), queries, dim3(256), 0, st, c, a, w, p.splits, p.chunk);
      if (p.splits > 1) hipLaunchKernelGGL(weigh_merge_kernel, dim3((rhos + 255) / 256, pairs), dim3(256), 0, st, c, a, w, p.splits, p.chunk, Q);
      if (p.ks == KS) hipLaunchKernelGGL((weigh_add_kernel<T, E, KS>), keys, dim3(256), 0, st, c, a, w, p.per, p.slices);
      else hipLaunchKernelGGL((weigh_add_kernel<T, E, 1>), keys, dim3(256), 0, st, c, a, w, p.per, p.slices);
      if (p.slices > 1)
        hipLaunchKernelGGL(weigh_sum_kernel, dim3((c.cap + 255) / 256, pairs), dim3(256), 0, st, c, a, w, p.per, 64 * p.ks, tile_rows<T, 16 * E>());
      MI_HIP(hipGetLastError());
      return MI_OK;
    });
  });
}

int launch_bounded_evict(const BoundedCache& c, int budget, int keep_first, int keep_last, void* ws, hipStream_t st) {
  if (budget >= c.cap) return MI_OK;                     // no row can hold more
  const int most = std::min(budget, c.cap - budget);
  const bool on_chip = c.cap <= ON_CHIP, move = most <= MOVE_MOST;
  const size_t pairs = (size_t)c.rows * c.Hkv, counts = move ? 0 : up256(pairs * 4), moves = move ? 0 : up256(pairs * most * 8);
  const EvictWs w{(int32_t*)ws, (int2*)((char*)ws + counts), (uint32_t*)((char*)ws + counts + moves), most};
  const dim3 grid(c.Hkv, c.rows);
  const int pieces = c.D * (int)dtype_size(c.dtype) / 16;
  const size_t lds = on_chip ? ((size_t)c.cap + c.cap / 32 + 1) * 4 : 0;
  auto select = [&](auto kern) {
    // (always the same limit: calls on other caches may set it in between)
    if (lds > 48 * 1024) MI_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (ON_CHIP + ON_CHIP / 32 + 1) * 4));
    hipLaunchKernelGGL(kern, grid, dim3(1024), lds, st, c, budget, keep_first, keep_last, pieces, w);
    return (int)MI_OK;
  };
  MI_TRY(on_chip ? (move ? select(evict_select_kernel<true, true>) : select(evict_select_kernel<true, false>))
                 : (move ? select(evict_select_kernel<false, true>) : select(evict_select_kernel<false, false>)));
  if (!move) {
    const int groups = (int)std::max<int64_t>(1, std::min<int64_t>(64, ((int64_t)most * pieces + 1023) / 1024));
    hipLaunchKernelGGL(evict_move_kernel, dim3(groups, c.rows * c.Hkv), dim3(256), 0, st, c, budget, pieces, w);
  }
  MI_HIP(hipGetLastError());
  return MI_OK;
}

}  // namespace mi
