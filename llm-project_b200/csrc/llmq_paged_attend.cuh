// llmq_paged_attend.cuh - attention of one query row a sequence over a paged
// cache: one pass over keys and values with a running maximum and sum.
//
// What bounds it: the cache's bytes.  Every key and value is read once for its
// KV head's whole group of query heads (blocks of kBlock heads; a larger group
// reads the cache once a block).
//
// Work is counted in tiles of kTile positions of one (row, KV head, block of
// heads), laid end to end over rows, heads and positions; each CTA of a grid
// that fills the GPU takes an equal, contiguous share, wherever it begins and
// ends.  So one long row is split over all SMs, and ragged rows leave none
// idle.  A CTA that covers a row's head from end to end writes the output; the at
// most two shares that are cut (one at its beginning, one at its end) are left
// in the workspace and joined by k_attend_join, one block for each query head of a cut.
//
// In a CTA each warp owns a slice of every tile (kSlice positions) with its own
// ring of kStages slices in shared memory, filled by 16-byte asynchronous
// copies: warps run without barriers until a (row, head) ends and their
// partial results are joined.  Positions past the row, before its window or on
// a page outside the pool are filled with zeros and masked, so what memory
// holds there (NaN too) is never used.
//
// Measured, both kernels in a captured graph (a plain copy moves 6.46 TB/s on the same GPU),
// 32 query heads (the long row: 64) on 8 KV heads of 128; in brackets calls in turn under
// seconds of load:
//   64 f32 rows of about 2100 positions      185 us, 5.99 TB/s (209 us, 5.32)
//   61 bf16 rows of up to 8191 positions     189 us, 5.94 TB/s (199 us, 5.63)
//   64 f32 rows over bf16, 2112 positions    100 us, 5.53 TB/s
//   one f16 row of 131072 positions           98 us, 5.45 TB/s (101 us): 6.95 TB/s in the long
//     run and some 17 us that do not depend on the length (launch, prefix sums, the first
//     loads' latency, the join)
//   8 bf16 rows of 512, 1024, 2048 positions  15, 18, 22 us, for 2.6, 5.2, 10.4 at the copy's rate
//   one row of a few hundred positions         7 us, the same chain without the bytes
//   16 bf16 rows of 4096, 16 query heads a KV head: 51 us, two readings of the 135 MB (20.8 for
//     one at the copy's rate)
// Counters at 16 rows of 2100: the cache read once (280 MB of DRAM reads for 278 MB), 42%
// (f32) and 33% (bf16) of the issue slots, 2 CTAs of 4 warps an SM (180 and 207
// registers): the ring, not the warps, keeps the memory busy.
// (One warp a row and head, plain loads and no split took 1794, 5016 and 57126 us.)
#pragma once

#include <climits>
#include <type_traits>

#include "llmq_serve.cuh"

namespace llmq {

struct AttendArgs {
  LlmqPagedKV kv;
  LlmqPagedAttention a;
  int row0, rows;      // the rows of this launch
  int blocks;          // blocks of heads a KV head
  float scale_log2;    // scale * log2(e)
  // position / page_size, for positions below 2^31: mulhi(position, div_mul) >> div_shift
  uint32_t div_mul;
  int div_shift;       // below 0: page_size 1
  long long page_bytes, token_bytes, head_bytes;  // the pool's strides
};

inline void set_division(AttendArgs &p) {
  const uint32_t d = static_cast<uint32_t>(p.kv.page_size);
  int l = 0;
  while ((1u << l) < d) ++l;  // 2^(l - 1) < d <= 2^l
  p.div_shift = l - 1;
  p.div_mul = l ? static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d) : 0;
}
__device__ __forceinline__ int page_of(const AttendArgs &p, int pos) {
  return p.div_shift < 0 ? pos : static_cast<int>(__umulhi(static_cast<uint32_t>(pos), p.div_mul) >> p.div_shift);
}

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kAttendStages = 3;
constexpr int kAttendMaxRows = 1024;  // rows of one launch
constexpr int kHeadBlock = 8;         // query heads of a partial result
// Units of a head beside its tiles: what joining the warps and fetching the next query
// cost, about two tiles' time.  Ragged bf16 rows of up to 8191 positions: 204 us without,
// 192 with one, 184 with two or three; 150 rows of up to 1000: 95, 77, 68, 69 us.
constexpr int kLead = 2;

// ------------------------------------------------------------- workspace
// For each CTA a header (the head it must join with earlier CTAs, if any) and two
// partial results of kHeadBlock heads: reference m, sum l, then head_dim sums.
struct JoinHeader {
  int row, kvh, block;  // row -1: nothing to join here
  int first, last;      // the CTAs whose partial results make it up
  int pad[3];
};
__host__ __device__ inline size_t attend_partial_floats(int hd) { return (size_t)kHeadBlock * (hd + 2); }
constexpr int kAttendMaxCtas = 640;  // four on each of 160 SMs
inline size_t attend_workspace(int hd) {
  return (size_t)kAttendMaxCtas * (sizeof(JoinHeader) + 2 * attend_partial_floats(hd) * sizeof(float));
}

// ---------------------------------------------------------------- pieces
__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes to shared memory; zeros when !valid (src is not read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r, x = *reinterpret_cast<unsigned long long *>(&a), y = *reinterpret_cast<unsigned long long *>(&b),
                        z = *reinterpret_cast<unsigned long long *>(&c);
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return *reinterpret_cast<float2 *>(&r);
}

// Of a reference m and the sum of 2^(s - m): 1 / sum and ln of what it stands for.  A sum of 0
// is a head without positions; a NaN (of a NaN or +infinite score) goes on into both.
__device__ __forceinline__ float share_of(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }
__device__ __forceinline__ float lse_of(float m, float sum) {
  return sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.693147180559945309f;
}

// What one row attends: positions [n0, n) in tiles [t0, t0 + tiles).
struct RowSpan {
  long long seq;
  int n0, n, t0, tiles;
};
__device__ __forceinline__ RowSpan row_span(const AttendArgs &p, int r, int tile, int *flags) {
  const LlmqPagedAttention &a = p.a;
  RowSpan s;
  s.seq = a.seqs ? a.seqs[r] : r;
  s.n = a.lens[r];
  const int cap = a.max_pages * p.kv.page_size;
  if (s.n < 0 || s.n > cap) {
    *flags |= LLMQ_PAGED_BAD_LEN;
    s.n = s.n < 0 ? 0 : cap;
  }
  if (s.seq < 0 || s.seq >= a.n_seqs) {
    if (s.n > 0) *flags |= LLMQ_PAGED_BAD_LEN;
    s.n = 0;
  }
  s.n0 = a.window > 0 && s.n > a.window ? s.n - a.window : 0;
  s.t0 = s.n0 / tile;
  s.tiles = s.n > 0 ? (s.n - 1) / tile + 1 - s.t0 : 0;
  return s;
}

// The partial result of one warp or CTA in shared memory: [kHeadBlock] rows of
// `pitch` sums, then m and l.
template <int HDP>
struct PartialBuf {
  static constexpr int kPitch = HDP + 4;  // a fragment's 4 x 8 elements (head 2 t, dim g) hit distinct banks
  static constexpr int kBytes = (kHeadBlock * kPitch + 2 * kHeadBlock) * 4;
  float *p;
  __device__ __forceinline__ float &o(int h, int d) const { return p[h * kPitch + d]; }
  __device__ __forceinline__ float &m(int h) const { return p[kHeadBlock * kPitch + h]; }
  __device__ __forceinline__ float &l(int h) const { return p[kHeadBlock * kPitch + kHeadBlock + h]; }
};

// ---------------------------------------------------- core for f32 pools
// Multiplications on the CUDA cores, two f32 at a time (fma.rn.f32x2): exact f32
// products.  kLanes lanes share a key, each with kDims of its dims; the lanes'
// partial scores of 32 / GB keys and GB heads are summed by a transposing
// reduction (31 exchanges for 32 scores), which leaves each lane one (key, head).
template <int HDP, int GB>
struct CoreF32 {
  typedef float Elem;
  typedef float Row;
  static constexpr int kBlock = GB;
  static constexpr int kSlice = 8;
  static constexpr int kLanes = HDP >= 128 ? 32 : HDP / 4, kGroups = 32 / kLanes;
  static constexpr int kQuads = HDP / 4 / kLanes;   // float4s of a row a lane owns
  static constexpr int kBatch = 32 / GB;            // keys scored at a time
  static constexpr int kPerGroup = kBatch / kGroups;
  static constexpr int kPitch = HDP * 4;            // bytes of a row in shared memory
  static constexpr int kSide = kSlice * GB * 8;     // the weights, each twice (a packed pair)
  static_assert(kSlice % kBatch == 0, "whole batches");
  float2 q[GB][2 * kQuads], o[GB][2 * kQuads];
  float m, l;  // of head lane % GB (m over all keys, l over the lane's)

  __device__ __forceinline__ void reset() {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int h = 0; h < GB; ++h)
#pragma unroll
      for (int i = 0; i < 2 * kQuads; ++i) o[h][i] = make_float2(0.0f, 0.0f);
  }
  __device__ __forceinline__ void load_q(const float *src, int nh, int hd, float) {
    const int lane = threadIdx.x & 31, c = lane % kLanes;
#pragma unroll
    for (int h = 0; h < GB; ++h)
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        const int d = 4 * (c + kLanes * i);  // head_dim % 8 == 0: a quad is whole or absent
        const float *s = src + (size_t)h * hd + d;
        const bool in = h < nh && d < hd;
        q[h][2 * i] = in ? make_float2(s[0], s[1]) : make_float2(0.0f, 0.0f);
        q[h][2 * i + 1] = in ? make_float2(s[2], s[3]) : make_float2(0.0f, 0.0f);
      }
  }
  // Adds a slice: keys at `buf`, values behind them; bit i of mask: key i counts.
  __device__ __forceinline__ void add(const char *buf, char *side, uint32_t mask, float scale_log2) {
    const int lane = threadIdx.x & 31, c = lane % kLanes, grp = lane / kLanes;
    float2 *w = reinterpret_cast<float2 *>(side);  // [kSlice][GB]
    float s[kSlice / kBatch];
    float mx = m;
#pragma unroll
    for (int b = 0; b < kSlice / kBatch; ++b) {
      float v[kLanes];
#pragma unroll
      for (int kb = 0; kb < kPerGroup; ++kb) {
        const char *row = buf + (size_t)(b * kBatch + grp * kPerGroup + kb) * kPitch;
        float2 k[2 * kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const float4 x = *reinterpret_cast<const float4 *>(row + 16 * (c + kLanes * i));
          k[2 * i] = make_float2(x.x, x.y);
          k[2 * i + 1] = make_float2(x.z, x.w);
        }
#pragma unroll
        for (int h = 0; h < GB; ++h) {
          float2 d = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int i = 0; i < 2 * kQuads; ++i) d = fma2(q[h][i], k[i], d);
          v[kb * GB + h] = d.x + d.y;
        }
      }
#pragma unroll
      for (int st = kLanes / 2; st > 0; st /= 2) {
        const bool up = lane & st;
#pragma unroll
        for (int i = 0; i < st; ++i) {
          const float give = up ? v[i] : v[i + st], keep = up ? v[i + st] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, st);
        }
      }
      // lane: key b * kBatch + lane / GB, head lane % GB
      s[b] = (mask >> (b * kBatch + lane / GB)) & 1u ? v[0] * scale_log2 : -INFINITY;
      mx = fmaxf(mx, s[b]);
    }
#pragma unroll
    for (int st = GB; st < 32; st *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, st));
    const float ref = mx == -INFINITY ? 0.0f : mx;
    if (__any_sync(0xffffffffu, mx > m)) {
      const float f = exp2_approx(m - ref);
      l *= f;
#pragma unroll
      for (int h = 0; h < GB; ++h) {
        const float fh = __shfl_sync(0xffffffffu, f, h);
#pragma unroll
        for (int i = 0; i < 2 * kQuads; ++i) o[h][i] = make_float2(o[h][i].x * fh, o[h][i].y * fh);
      }
      m = mx;
    }
#pragma unroll
    for (int b = 0; b < kSlice / kBatch; ++b) {
      const float e = exp2_approx(s[b] - ref);
      l += e;
      w[(b * kBatch + lane / GB) * GB + lane % GB] = make_float2(e, e);
    }
    __syncwarp();
    const char *vals = buf + kSlice * kPitch;
#pragma unroll
    for (int b = 0; b < kSlice / kBatch; ++b)
#pragma unroll
      for (int kb = 0; kb < kPerGroup; ++kb) {
        const int key = b * kBatch + grp * kPerGroup + kb;
        float2 x[2 * kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const float4 y = *reinterpret_cast<const float4 *>(vals + (size_t)key * kPitch + 16 * (c + kLanes * i));
          x[2 * i] = make_float2(y.x, y.y);
          x[2 * i + 1] = make_float2(y.z, y.w);
        }
#pragma unroll
        for (int h = 0; h < GB; ++h) {
          const float2 e = w[key * GB + h];
#pragma unroll
          for (int i = 0; i < 2 * kQuads; ++i) o[h][i] = fma2(e, x[i], o[h][i]);
        }
      }
    __syncwarp();
  }
  __device__ __forceinline__ void write(const PartialBuf<HDP> &b) {
    const int lane = threadIdx.x & 31, c = lane % kLanes;
#pragma unroll
    for (int st = GB; st < 32; st *= 2) l += __shfl_xor_sync(0xffffffffu, l, st);
    if (lane < GB) {
      b.m(lane) = m;
      b.l(lane) = l;
    }
#pragma unroll
    for (int h = 0; h < GB; ++h)
#pragma unroll
      for (int i = 0; i < 2 * kQuads; ++i) {
        float2 x = o[h][i];
#pragma unroll
        for (int st = kLanes; st < 32; st *= 2) {
          x.x += __shfl_xor_sync(0xffffffffu, x.x, st);
          x.y += __shfl_xor_sync(0xffffffffu, x.y, st);
        }
        if (lane < kLanes)
          *reinterpret_cast<float2 *>(&b.o(h, 4 * (c + kLanes * (i / 2)) + 2 * (i % 2))) = x;
      }
  }
};

// -------------------------------------------------- core for 16-bit pools
// mma.sync m16n8k16 with the cache as the 16-row operand: scores^T = K q^T (16
// keys x 8 heads) and out^T = V^T w^T (16 dims x 8 heads), so 8 heads fill the
// instruction and no row is wasted; a slice of 16 keys of 128 dims is 8 KB of
// cache for 16 instructions a term, far below what the tensor cores do in the
// time the 8 KB take to arrive (372 cycles of an SM's share of the measured
// bandwidth), which is why the larger tcgen05 tiles (128 rows, a group has at
// most 8) would gain nothing here.
// The rows' elements multiply exactly: a 16-bit q is its own single term; an f32 q
// is scaled by a power of two (per head) and split into three 16-bit terms, and
// the weights are split into kW terms (bf16 8 bits, f16 11 bits each).
template <typename T, typename KT>
struct Terms {
  static constexpr bool kF16 = std::is_same<KT, __half>::value;
  static constexpr int kQ = std::is_same<T, float>::value ? 3 : 1;
  // f32 rows: 24 bits of bf16, 22 of f16 terms; 16-bit rows: 16 and 22 bits,
  // beyond the output's own 8 and 11
  static constexpr int kW = std::is_same<T, float>::value && !kF16 ? 3 : 2;
  // f16 weights lie in [0, 2^14], so that one 2^-24 of the largest is still normal
  static constexpr float kLift = kF16 ? 14.0f : 0.0f;
};

template <typename KT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename KT>
__device__ __forceinline__ float2 unpack16(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack16<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <>
__device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
}

template <typename KT>
__device__ __forceinline__ void mma16816(float *d, const uint32_t *a, const uint32_t *b) {
  if constexpr (std::is_same<KT, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <bool trans>
__device__ __forceinline__ void ldmatrix4(uint32_t *r, uint32_t addr) {
  if constexpr (trans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T, typename KT, int HDP>
struct CoreMma {
  typedef KT Elem;
  typedef T Row;
  typedef Terms<T, KT> Tm;
  static constexpr int kBlock = 8;
  static constexpr int kSlice = 16;
  static constexpr int kSteps = HDP / 16;
  static constexpr int kPitch = HDP * 2 + 16;  // an odd number of 16-byte pieces: ldmatrix rows hit distinct banks
  static constexpr int kSide = 0;
  uint32_t q[Tm::kQ][kSteps][2];
  float o[kSteps][4];  // dims 16 i + g and + 8, heads 2 t and 2 t + 1 (lane = 4 g + t)
  float m[2], l[2], sc[2];

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[j] = -INFINITY;
      l[j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
  }
  __device__ __forceinline__ void load_q(const T *src, int nh, int hd, float scale_log2) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (Tm::kQ == 1) {
      sc[0] = sc[1] = scale_log2;
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = 16 * i + 8 * j + 2 * t;  // head_dim % 8 == 0: both dims exist or neither
          const KT *s = src + (size_t)g * hd + d;
          const bool in = g < nh && d < hd;
          q[0][i][j] = in ? pack16<KT>(to_f32(s[0]), to_f32(s[1])) : 0u;
        }
    } else {
      float2 x[kSteps][2];
      float big = 0.0f;
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = 16 * i + 8 * j + 2 * t;
          const T *s = src + (size_t)g * hd + d;
          x[i][j] = g < nh && d < hd ? make_float2(s[0], s[1]) : make_float2(0.0f, 0.0f);
          big = fmaxf(big, fmaxf(fabsf(x[i][j].x), fabsf(x[i][j].y)));
        }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // the head's largest element to [2^14, 2^15): every term is a normal number
      const int e = big > 0.0f && big < INFINITY ? min(max(ilogbf(big) - 14, -120), 120) : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float2 r = make_float2(x[i][j].x * down, x[i][j].y * down);
#pragma unroll
          for (int n = 0; n < Tm::kQ; ++n) {
            q[n][i][j] = pack16<KT>(r.x, r.y);
            const float2 h = unpack16<KT>(q[n][i][j]);
            r = make_float2(r.x - h.x, r.y - h.y);
          }
        }
      const float mine = scale_log2 * up;  // of head g
      sc[0] = __shfl_sync(0xffffffffu, mine, 8 * t);
      sc[1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
    }
  }
  __device__ __forceinline__ void add(const char *buf, char *, uint32_t mask, float) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const uint32_t base = smem_addr(buf);
    // rows of the four 8 x 8 pieces of a step: keys (lane & 15), dims 8 (lane >> 4)
    const uint32_t ka = base + (lane & 15) * kPitch + (lane >> 4) * 16;
    float s[2][4] = {};  // two chains over the steps
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      uint32_t a[4];
      ldmatrix4<false>(a, ka + 32 * i);
#pragma unroll
      for (int n = Tm::kQ - 1; n >= 0; --n) mma16816<KT>(s[i & 1], a, q[n][i]);
    }
    float mx[2] = {m[0], m[1]}, v[2][2];  // [key g, g + 8][head 2 t, 2 t + 1]
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v[k][j] = (mask >> (g + 8 * k)) & 1u ? (s[0][2 * k + j] + s[1][2 * k + j]) * sc[j] : -INFINITY;
        mx[j] = fmaxf(mx[j], v[k][j] - Tm::kLift);
      }
#pragma unroll
    for (int st = 4; st < 32; st *= 2)
#pragma unroll
      for (int j = 0; j < 2; ++j) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], st));
    float ref[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) ref[j] = mx[j] == -INFINITY ? 0.0f : mx[j];
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
      const float f0 = exp2_approx(m[0] - ref[0]), f1 = exp2_approx(m[1] - ref[1]);
      l[0] *= f0;
      l[1] *= f1;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        o[i][0] *= f0;
        o[i][1] *= f1;
        o[i][2] *= f0;
        o[i][3] *= f1;
      }
      m[0] = mx[0];
      m[1] = mx[1];
    }
    uint32_t w[Tm::kW][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float2 r = make_float2(exp2_approx(v[k][0] - ref[0]), exp2_approx(v[k][1] - ref[1]));
      l[0] += r.x;
      l[1] += r.y;
#pragma unroll
      for (int n = 0; n < Tm::kW; ++n) {
        const uint32_t x = pack16<KT>(r.x, r.y);
        const float2 h = unpack16<KT>(x);
        r = make_float2(r.x - h.x, r.y - h.y);
        w[n][k] = transpose8x8(x);  // from [key][head] to the operand's [head][key]
      }
    }
    // values transposed on the way: dims 8 ((lane >> 3) & 1), keys (lane & 7) + 8 (lane >> 4)
    const uint32_t va = base + kSlice * kPitch + ((lane & 7) + (lane >> 4) * 8) * kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      uint32_t a[4];
      ldmatrix4<true>(a, va + 32 * i);
#pragma unroll
      for (int n = Tm::kW - 1; n >= 0; --n) mma16816<KT>(o[i], a, w[n]);
    }
  }
  __device__ __forceinline__ void write(const PartialBuf<HDP> &b) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int st = 4; st < 32; st *= 2)
#pragma unroll
      for (int j = 0; j < 2; ++j) l[j] += __shfl_xor_sync(0xffffffffu, l[j], st);
    if (g == 0)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        b.m(2 * t + j) = m[j];
        b.l(2 * t + j) = l[j];
      }
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) b.o(2 * t + (j & 1), 16 * i + g + 8 * (j >> 1)) = o[i][j];
  }
};

// --------------------------------------------------------------- kernels
template <typename Core, int HDP>
struct AttendShape {
  static constexpr int kTile = Core::kSlice * kAttendWarps;
  static constexpr int kStage = 2 * Core::kSlice * Core::kPitch;
  static constexpr int kSmem = kAttendWarps * (kAttendStages * kStage + Core::kSide);
  // CTAs of an SM: what its shared memory holds, at most 4
  static constexpr int kFit = (224 * 1024) / (kSmem + 2048);
  static constexpr int kPerSm = kFit < 4 ? kFit : 4;
  static_assert(kPerSm >= 1, "a CTA fits an SM");
  static_assert(kStage >= PartialBuf<HDP>::kBytes, "a partial result fits a stage");
  static_assert(kStage % 16 == 0 && Core::kSide % 16 == 0, "16-byte pieces");
};

// A place in the CTA's share: row, KV head, block of heads, tile.
struct Cursor {
  RowSpan span;
  int row, kvh, block, tile;
  long long unit;
};

template <typename Core, int HDP>
__global__ void __launch_bounds__(kAttendThreads, AttendShape<Core, HDP>::kPerSm) k_attend(const AttendArgs p) {
  typedef AttendShape<Core, HDP> Sh;
  typedef typename Core::Elem KT;
  typedef typename Core::Row T;
  constexpr int kSlice = Core::kSlice, kLpr = HDP * (int)sizeof(KT) / 16 <= 8    ? 8
                                             : HDP * (int)sizeof(KT) / 16 <= 16 ? 16
                                                                                : 32;
  constexpr int kPieces = 16 / sizeof(KT);                                // elements of a 16-byte piece
  constexpr int kRounds = (HDP / kPieces + kLpr - 1) / kLpr;              // pieces of a row a lane copies
  extern __shared__ __align__(128) char s_ring[];
  __shared__ uint32_t s_mask[kAttendWarps][kAttendStages];
  __shared__ float s_factor[kAttendWarps][kHeadBlock], s_inv[kHeadBlock];
  __shared__ long long s_sum[kAttendWarps], s_rows[kAttendWarps];
  __shared__ long long s_base;
  __shared__ int s_row;
  const LlmqPagedKV &kv = p.kv;
  const LlmqPagedAttention &a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = kv.head_dim;
  char *ring = s_ring + (size_t)warp * (kAttendStages * Sh::kStage + Core::kSide);
  char *side = ring + kAttendStages * Sh::kStage;
  // dims past head_dim stay zero
  if (hd < HDP) for (int i = lane * 16; i < kAttendStages * Sh::kStage; i += 512) *reinterpret_cast<int4 *>(ring + i) = make_int4(0, 0, 0, 0);
  serve_wait();
  serve_dependents();

  // ---- this CTA's share: units [x0, x1).  A head takes a unit a tile, after `lead` units
  // for what its end costs beside its tiles (joining the warps, the next head's query)
  const int per_row = kv.n_kv * p.blocks, each = (p.rows + kAttendThreads - 1) / kAttendThreads;
  const int ra = p.row0 + min(p.rows, tid * each), rb = p.row0 + min(p.rows, (tid + 1) * each);
  int flags = 0;
  long long mine = 0, mine_rows = 0;
  for (int r = ra; r < rb; ++r) {
    const int n = row_span(p, r, Sh::kTile, &flags).tiles;
    mine += n;
    mine_rows += n > 0;
  }
  const bool empty = __syncthreads_or(mine_rows < rb - ra);  // some row has no position
  if (blockIdx.x == 0 && flags && a.status) atomicOr(a.status, flags);
  flags = 0;
  long long incl = mine, incl_rows = mine_rows;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, incl, o), v = __shfl_up_sync(0xffffffffu, incl_rows, o);
    if (lane >= o) {
      incl += u;
      incl_rows += v;
    }
  }
  if (lane == 31) {
    s_sum[warp] = incl;
    s_rows[warp] = incl_rows;
  }
  __syncthreads();
  long long total = 0, rows_total = 0, before = incl - mine, rows_before = incl_rows - mine_rows;
  for (int w = 0; w < kAttendWarps; ++w) {
    if (w < warp) {
      before += s_sum[w];
      rows_before += s_rows[w];
    }
    total += s_sum[w];
    rows_total += s_rows[w];
  }
  // with only a few tiles a CTA the tiles themselves are spread as evenly as they can be
  const int lead = total * per_row > 4LL * gridDim.x ? kLead : 0;
  total = (total + lead * rows_total) * per_row;
  before += lead * rows_before;
  mine += lead * mine_rows;
  const long long ctas = min(static_cast<long long>(gridDim.x), total);  // none has an empty share
  const bool idle = blockIdx.x >= ctas;
  const long long x0 = idle ? total : blockIdx.x * total / ctas, x1 = idle ? total : (blockIdx.x + 1) * total / ctas;
  if (before * per_row <= x0 && x0 < (before + mine) * per_row) {
    int ignored = 0;
    for (int r = ra; r < rb; ++r) {
      const int t = row_span(p, r, Sh::kTile, &ignored).tiles, n = t ? t + lead : 0;
      if (x0 < (before + n) * per_row) {
        s_row = r;
        s_base = before;
        break;
      }
      before += n;
    }
  }
  JoinHeader *headers = static_cast<JoinHeader *>(a.workspace);
  float *partials = reinterpret_cast<float *>(headers + gridDim.x);
  const size_t psize = attend_partial_floats(hd);
  __syncthreads();
  if (tid == 0) headers[blockIdx.x].row = -1;
  auto empty_rows = [&]() {
    if (!empty) return;
    for (int r = p.row0 + blockIdx.x; r < p.row0 + p.rows; r += gridDim.x) {
      int ignored = 0;
      if (row_span(p, r, Sh::kTile, &ignored).tiles == 0) {
        for (int e = tid; e < a.n_heads * hd; e += kAttendThreads)
          static_cast<T *>(a.out)[r * a.out_stride + e] = from_f32<T>(0.0f);
        for (int h = tid; h < a.n_heads && a.lse; h += kAttendThreads) a.lse[(size_t)r * a.n_heads + h] = -INFINITY;
      }
    }
  };
  if (x0 >= x1) {
    empty_rows();
    return;
  }

  Cursor in;  // the next slice to fetch
  in.row = s_row;
  {
    int ignored = 0;
    in.span = row_span(p, in.row, Sh::kTile, &ignored);
  }
  {
    const long long rel = x0 - s_base * per_row, size = in.span.tiles + lead;
    const int pair = static_cast<int>(rel / size), in_pair = static_cast<int>(rel - pair * size);
    in.tile = max(0, in_pair - lead);
    in.unit = x0 - in_pair + lead + in.tile;
    in.kvh = pair / p.blocks;
    in.block = pair - in.kvh * p.blocks;
  }
  if (in.unit >= x1) {  // a share of lead units alone
    empty_rows();
    return;
  }
  Cursor at = in;  // the slice to add
  auto advance = [&](Cursor &c) {
    ++c.unit;
    if (++c.tile < c.span.tiles) return;
    c.tile = 0;
    c.unit += lead;
    if (++c.block < p.blocks) return;
    c.block = 0;
    if (++c.kvh < kv.n_kv) return;
    c.kvh = 0;
    int ignored = 0;
    do {
      if (++c.row >= p.row0 + p.rows) return;  // past the share: not used
      c.span = row_span(p, c.row, Sh::kTile, &ignored);
    } while (c.span.tiles == 0);
  };
  // Keys are looked up by runs of 8, which a page of a multiple of 8 positions does not
  // split: a lane each, the next slice's while this one's copies are issued.  Other
  // page sizes take a lookup a key.
  const bool runs = kv.page_size % 8 == 0;
  const int lookups = runs ? kSlice / 8 : kSlice, run = runs ? 8 : 1;
  int page = -1, within = 0;  // of the lane's run: its page, the first key's place in it
  bool asked = false;
  auto find_page = [&]() {
    const int pos = (in.span.t0 + in.tile) * Sh::kTile + warp * kSlice + lane * run;
    page = -1;
    asked = false;
    if (lane < lookups && pos + run > in.span.n0 && pos < in.span.n) {
      const int i = page_of(p, pos);
      within = pos - i * kv.page_size;
      page = a.table[in.span.seq * a.table_stride + i];  // looked at in the next fetch: no wait here
      asked = true;
    }
  };
  bool more = true;  // slices to fetch
  int put = 0;
  find_page();
  const int group = a.n_heads / kv.n_kv;
  Core core;
  auto load_q = [&](const Cursor &c) {
    const int h0 = c.kvh * group + c.block * Core::kBlock;
    core.load_q(static_cast<const T *>(a.q) + c.row * a.q_stride + (size_t)h0 * hd, min(Core::kBlock, group - c.block * Core::kBlock),
                hd, p.scale_log2);
  };
  load_q(at);  // on its way with the lookup
  core.reset();
  constexpr int kRows = 32 / kLpr;  // rows a round of copies covers
  const int piece = lane % kLpr;
  const bool copies = piece * kPieces < hd;
  const long long lane_bytes = (lane / kLpr) * p.token_bytes + piece * 16, round_bytes = kRows * p.token_bytes;
  const long long to_v = static_cast<const char *>(kv.v) - static_cast<const char *>(kv.k);
  auto fetch = [&]() {
    if (more) {
      const int base = (in.span.t0 + in.tile) * Sh::kTile + warp * kSlice;
      // keys [n0, n) of the slice, less those without a page
      const int lo = min(max(in.span.n0 - base, 0), kSlice), hi = min(max(in.span.n - base, 0), kSlice);
      uint32_t mask = (0xffffffffu >> 1 >> (31 - hi)) & ~((1u << lo) - 1u);
      const bool good = asked && static_cast<unsigned>(page) < static_cast<unsigned>(kv.n_pages);
      if (asked && !good) flags |= LLMQ_PAGED_BAD_PAGE;
      uint32_t have = __ballot_sync(0xffffffffu, good);
      if (runs) have = (have & 1u ? 0xffu : 0u) | (have & 2u ? 0xff00u : 0u);
      mask &= have;
      if (lane == 0) s_mask[warp][put] = mask;
      if (mask) {
        const long long off = good ? page * p.page_bytes + within * p.token_bytes : 0;
        const char *kb = static_cast<const char *>(kv.k) + in.kvh * p.head_bytes;
        const uint32_t dst = smem_addr(ring + put * Sh::kStage) + (lane / kLpr) * Core::kPitch + piece * 16;
        auto copy_row = [&](uint32_t d, const char *src, bool all, bool ok) {
          if (!copies) return;
#pragma unroll
          for (int i = 0; i < kRounds; ++i)
            if (i == 0 || (piece + i * kLpr) * kPieces < hd) {
              const char *k = src + i * kLpr * 16;
              if (all) {
                copy16(d + i * kLpr * 16, k);
                copy16(d + i * kLpr * 16 + kSlice * Core::kPitch, k + to_v);
              } else {
                copy16(d + i * kLpr * 16, k, ok);
                copy16(d + i * kLpr * 16 + kSlice * Core::kPitch, k + to_v, ok);
              }
            }
        };
        if (runs) {
#pragma unroll
          for (int g = 0; g < kSlice / 8; ++g) {
            const char *src = kb + __shfl_sync(0xffffffffu, off, g) + lane_bytes;
            const bool all = ((mask >> (8 * g)) & 0xffu) == 0xffu;
#pragma unroll
            for (int it = 0; it < 8 / kRows; ++it) {
              const int row = 8 * g + it * kRows;
              copy_row(dst + row * Core::kPitch, src, all, (mask >> (row + lane / kLpr)) & 1u);
              src += round_bytes;
            }
          }
        } else {
#pragma unroll
          for (int it = 0; it < kSlice / kRows; ++it) {
            const int row = it * kRows + lane / kLpr;
            const char *src = kb + __shfl_sync(0xffffffffu, off, row) + piece * 16;
            copy_row(dst + it * kRows * Core::kPitch, src, false, (mask >> row) & 1u);
          }
        }
      }
      put = put + 1 == kAttendStages ? 0 : put + 1;
      advance(in);
      more = in.unit < x1;
      if (more) find_page();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  bool fresh = false, whole = at.tile == 0;  // whole: the share has this head from its first tile
  int get = 0;
#pragma unroll
  for (int i = 0; i < kAttendStages - 1; ++i) fetch();
  empty_rows();
  while (true) {
    const int h0 = at.kvh * group + at.block * Core::kBlock;
    const int nh = min(Core::kBlock, group - at.block * Core::kBlock);
    if (fresh) {
      core.reset();
      load_q(at);
      fresh = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kAttendStages - 2) : "memory");
    __syncwarp();
    const uint32_t mask = s_mask[warp][get];
    if (mask) core.add(ring + get * Sh::kStage, side, mask, p.scale_log2);
    const bool ends = at.tile + 1 == at.span.tiles;
    if (ends || at.unit + 1 == x1) {
      // ---- the head, or the share's part of it, is done: join the warps
      __syncwarp();
      core.write(PartialBuf<HDP>{reinterpret_cast<float *>(ring + get * Sh::kStage)});
      __syncthreads();
      auto of = [&](int w) {
        return PartialBuf<HDP>{reinterpret_cast<float *>(s_ring + (size_t)w * (kAttendStages * Sh::kStage + Core::kSide) +
                                                         get * Sh::kStage)};
      };
      const bool out_now = ends && whole;
      float *part = partials + (2 * (size_t)blockIdx.x + (whole ? 1 : 0)) * psize;
      if (tid < kHeadBlock) {  // a thread a head: the warps' factors
        const int h = tid;
        float mx = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) mx = h < nh ? fmaxf(mx, of(w).m(h)) : mx;
        const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) {
          const float f = h < nh ? exp2_approx(of(w).m(h) - ref) : 0.0f;
          sum += h < nh ? of(w).l(h) * f : 0.0f;
          s_factor[w][h] = f;
        }
        s_inv[h] = out_now ? share_of(sum) : 1.0f;
        if (h < nh) {
          if (!out_now) {
            part[h] = mx;
            part[kHeadBlock + h] = sum;
          } else if (a.lse) {
            a.lse[(size_t)at.row * a.n_heads + h0 + h] = lse_of(mx, sum);
          }
        }
      }
      __syncthreads();
      const bool out16 = out_now && (reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(T)) == 0) && a.out_stride % 4 == 0;
#pragma unroll 2
      for (int e = tid; e < nh * (hd / 4); e += kAttendThreads) {
        const int h = e / (hd / 4), d = 4 * (e - h * (hd / 4));
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) {
          const float f = s_factor[w][h];
          const float4 x = *reinterpret_cast<const float4 *>(&of(w).o(h, d));
          v.x = fmaf(x.x, f, v.x);
          v.y = fmaf(x.y, f, v.y);
          v.z = fmaf(x.z, f, v.z);
          v.w = fmaf(x.w, f, v.w);
        }
        const float inv = s_inv[h];
        if (out_now) {
          T *o = static_cast<T *>(a.out) + at.row * a.out_stride + (size_t)(h0 + h) * hd + d;
          const Pack<T, 4> y{{from_f32<T>(v.x * inv), from_f32<T>(v.y * inv), from_f32<T>(v.z * inv), from_f32<T>(v.w * inv)}};
          if (out16) {
            *reinterpret_cast<Pack<T, 4> *>(o) = y;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = y.v[i];
          }
        } else {
          *reinterpret_cast<float4 *>(part + 2 * kHeadBlock + h * hd + d) = v;
        }
      }
      if (!whole && tid == 0) {
        // this CTA begins inside the head: the second CTA of the head sees to the join
        const long long g0 = at.unit - at.tile, g1 = g0 + at.span.tiles;
        const long long first = ((g0 + 1) * ctas - 1) / total, last = (g1 * ctas - 1) / total;
        if (first + 1 == blockIdx.x) {
          JoinHeader h{};
          h.row = at.row;
          h.kvh = at.kvh;
          h.block = at.block;
          h.first = static_cast<int>(first);
          h.last = static_cast<int>(last);
          headers[blockIdx.x] = h;
        }
      }
      __syncthreads();
      // dims past head_dim of the stage: zero again
      if (hd < HDP) for (int i = lane * 16; i < Sh::kStage; i += 512)
        *reinterpret_cast<int4 *>(ring + get * Sh::kStage + i) = make_int4(0, 0, 0, 0);
      fresh = whole = true;
    }
    __syncwarp();
    get = get + 1 == kAttendStages ? 0 : get + 1;
    advance(at);
    if (at.unit >= x1) break;
    fetch();
  }
  if (flags && a.status) atomicOr(a.status, flags);
}

// Joins the partial results of a head that CTAs first .. last of a header share:
// block (header, head of its block), a thread four dims of every kth partial result, so
// that a long row's few dozen are read in one or two rounds of loads.
constexpr int kJoinThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) k_attend_join(const AttendArgs p, int ctas, int head_block) {
  __shared__ float s_f[kAttendMaxCtas];  // factors of the partial results
  __shared__ float4 s_v[kJoinThreads];
  __shared__ float s_red[2][kJoinThreads / 32];
  serve_wait();
  serve_dependents();
  const LlmqPagedAttention &a = p.a;
  const JoinHeader *headers = static_cast<const JoinHeader *>(a.workspace);
  const JoinHeader at = headers[blockIdx.x];
  const int hd = p.kv.head_dim, group = a.n_heads / p.kv.n_kv, h = blockIdx.y;
  if (at.row < 0 || at.block * head_block + h >= group) return;
  const int n = at.last - at.first + 1, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t psize = attend_partial_floats(hd);
  // the first CTA has it as the end of its share, the others as the beginning
  const float *partials = reinterpret_cast<const float *>(headers + ctas) + 2 * (size_t)at.first * psize;
  auto of = [&](int c) { return partials + (2 * (size_t)c + (c == 0 ? 1 : 0)) * psize; };
  constexpr int kMine = (kAttendMaxCtas + kJoinThreads - 1) / kJoinThreads;
  float m[kMine], l[kMine], mx = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int c = tid + i * kJoinThreads;
    m[i] = c < n ? of(c)[h] : -INFINITY;
    l[i] = c < n ? of(c)[kHeadBlock + h] : 0.0f;
    mx = fmaxf(mx, m[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) s_red[0][warp] = mx;
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 32; ++w) mx = fmaxf(mx, s_red[0][w]);
  const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int c = tid + i * kJoinThreads;
    const float f = exp2_approx(m[i] - ref);
    sum += l[i] * f;
    if (c < n) s_f[c] = f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_red[1][warp] = sum;
  __syncthreads();
  sum = 0.0f;
  for (int w = 0; w < kJoinThreads / 32; ++w) sum += s_red[1][w];
  const int pieces = hd / 4;  // at most 64
  const int groups = kJoinThreads / pieces, g = tid / pieces, d = 4 * (tid - g * pieces);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (g < groups) {
#pragma unroll 8
    for (int c = g; c < n; c += groups) {
      const float4 x = *reinterpret_cast<const float4 *>(of(c) + 2 * kHeadBlock + h * hd + d);
      const float f = s_f[c];
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
      v.z = fmaf(x.z, f, v.z);
      v.w = fmaf(x.w, f, v.w);
    }
    s_v[tid] = v;
  }
  __syncthreads();
  const int head = at.kvh * group + at.block * head_block + h;
  if (g == 0) {
    for (int q = 1; q < min(groups, n); ++q) {
      const float4 x = s_v[q * pieces + tid];
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    const float inv = share_of(sum);
    T *o = static_cast<T *>(a.out) + at.row * a.out_stride + (size_t)head * hd + d;
    o[0] = from_f32<T>(v.x * inv);
    o[1] = from_f32<T>(v.y * inv);
    o[2] = from_f32<T>(v.z * inv);
    o[3] = from_f32<T>(v.w * inv);
  }
  if (tid == 0 && a.lse)
    a.lse[(size_t)at.row * a.n_heads + head] = lse_of(mx, sum);
}

}  // namespace llmq
