// What the attention kernels over paged K/V share: the problem, how its work is cut into equal spans, and the
// partial results that the merge kernel joins.
//
// Rows. The new tokens of a request times the G query heads of one KV head form q*G rows (row = token * G + head), so
// a K or V row is read once for all of them. A unit is a tile of consecutive rows of one (request, KV head) together
// with the keys its tokens see: keys [lo, hi) of token i at position p = kv_len - q + i,
//     lo = max(0, p - window + 1),   hi = min(kv_len, max(p + 1, prefix_len)),
// both growing with i, so a tile's range is its first token's lo to its last token's hi.
//
// Spans. Requests differ in length, and only the device knows how. The units' key tiles, laid end to end (request,
// KV head, row tile, key tile), are cut into one span per block of equal length, so every block has the same work
// whatever the mix. A unit that a cut divides leaves one partial (o, m, l) per piece, at a place that follows from
// the block's number: nothing is counted, nothing needs to be cleared before a call, and the pieces are always
// added in the same order. A cut that would fall within `snap` tiles of a unit's edge moves to the edge.
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>

namespace kvb {

constexpr int PA_MAX_B = 8192;
constexpr float PA_LOG2E = 1.4426950408889634f;
constexpr float PA_LN2 = 0.6931471805599453f;

struct PagedParams {
  const void* q; int64_t q_st, q_sh;                 // [N,Hq,D]
  const void* key; int64_t k_sp, k_sh, k_st;         // pools [num_pages,Hkv,P,D]
  const void* value; int64_t v_sp, v_sh, v_st;
  const int32_t* table; int64_t table_st; int W, shift, num_pages;
  const int32_t* cu_q;                               // [B+1] or NULL: one token per request
  const int32_t* kv_len;                             // [B]
  const int32_t* prefix;                             // [B] or NULL
  const float* slopes;                               // [Hq] or NULL
  int N, B, Hq, Hkv, G, window;
  float scale_log2;                                  // scaling * log2(e)
  float cap_in, cap_log2;                            // scaling / softcap, softcap * log2(e); cap_log2 == 0: none
  void* out;                                         // [N,Hq,D]
  float* lse;                                        // [N,Hq] or NULL
  float* ws_o;                                       // [2*grid][ROWS][D] un-normalised outputs of unit pieces
  float2* ws_ml;                                     // [2*grid][ROWS] (m, l)
  int4* ws_desc;                                     // [2*grid]: see PieceDesc
  int grid;
  int box;                                           // rows per TMA box of a pool, 0: no TMA
};

// ws_desc[2c]: the piece that continues a unit begun by an earlier block: x = 1, y = 1 iff the unit ends in it.
// ws_desc[2c+1]: the piece that begins a unit which a later block ends: x = 1, y = request, z = KV head, w = row tile.
// x = 0: no such piece.

struct PagedRequest {
  int first, q, kv, pre;      // first row of the packed query, new tokens, keys, prefix; position of token i: kv - q + i
};

__device__ __forceinline__ PagedRequest paged_request(const PagedParams& p, int b) {
  PagedRequest r;
  if (p.cu_q) {
    const int a = min(max(p.cu_q[b], 0), p.N), e = min(max(p.cu_q[b + 1], 0), p.N);
    r.first = a;
    r.q = max(e - a, 0);
  } else {
    r.first = b;
    r.q = 1;
  }
  const int64_t most = (int64_t)p.W << p.shift;
  r.kv = (int)min((int64_t)max(p.kv_len[b], 0), most);
  r.pre = p.prefix ? min(max(p.prefix[b], 0), r.kv) : 0;
  return r;
}
__device__ __forceinline__ int paged_lo(const PagedRequest& r, int window, int i) {
  return window > 0 ? max(0, r.kv - r.q + i - window + 1) : 0;
}
__device__ __forceinline__ int paged_hi(const PagedRequest& r, int i) { return min(r.kv, max(r.kv - r.q + i + 1, r.pre)); }

// The key range of row tile t (rows [t*ROWS, ...) of q*G) and its key tiles [t0, t1) of KT keys; a tile that sees no
// key still counts as one, so that its rows are written.
template <int ROWS, int KT>
struct PagedUnit {
  int lo, hi, t0, n;
  __device__ __forceinline__ void set(const PagedRequest& r, int G, int window, int tile) {
    const int i0 = tile * ROWS / G, i1 = min(r.q - 1, (tile * ROWS + ROWS - 1) / G);
    lo = paged_lo(r, window, i0);
    hi = max(paged_hi(r, i1), 0);
    if (hi <= lo) { lo = hi = 0; }
    t0 = lo / KT;
    n = max(1, (hi + KT - 1) / KT - t0);
  }
};
template <int ROWS>
__device__ __forceinline__ int paged_row_tiles(const PagedRequest& r, int G) {
  return (int)(((int64_t)r.q * G + ROWS - 1) / ROWS);
}

struct PagedPlace { int b, h, tile, k; };            // a key tile: request, KV head, row tile, key tile of the unit

// Cuts the work. Called by every thread of the block; s_sum: B words of shared memory, free again afterwards.
// Returns the block's first key tile and how many it has.
template <int ROWS, int KT, int THREADS>
__device__ __forceinline__ void paged_span(const PagedParams& p, int* s_sum, PagedPlace& place, long long& count, int snap) {
  __shared__ long long s_total;
  __shared__ PagedPlace s_place[2];
  __shared__ long long s_pos[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WARPS = THREADS / 32;
  // key tiles of one KV head of every request
  for (int b0 = warp * 32; b0 < p.B; b0 += WARPS * 32) {
    const int b = b0 + lane;
    PagedRequest r = {0, 0, 0, 0};
    int tiles = 0, sum = 0;
    if (b < p.B) {
      r = paged_request(p, b);
      tiles = paged_row_tiles<ROWS>(r, p.G);
      if (tiles <= 4)
        for (int t = 0; t < tiles; ++t) {
          PagedUnit<ROWS, KT> u;
          u.set(r, p.G, p.window, t);
          sum += u.n;
        }
    }
    unsigned big = __ballot_sync(0xffffffffu, tiles > 4);
    while (big) {
      const int src = __ffs(big) - 1;
      big &= big - 1;
      const PagedRequest rr = {__shfl_sync(0xffffffffu, r.first, src), __shfl_sync(0xffffffffu, r.q, src),
                               __shfl_sync(0xffffffffu, r.kv, src), __shfl_sync(0xffffffffu, r.pre, src)};
      const int nt = __shfl_sync(0xffffffffu, tiles, src);
      int part = 0;
      for (int t = lane; t < nt; t += 32) {
        PagedUnit<ROWS, KT> u;
        u.set(rr, p.G, p.window, t);
        part += u.n;
      }
      part = __reduce_add_sync(0xffffffffu, part);
      if (lane == src) sum = part;
    }
    if (b < p.B) s_sum[b] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    long long t = 0;
    for (int b = lane; b < p.B; b += 32) t += s_sum[b];
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    if (lane == 0) s_total = t * p.Hkv;
  }
  __syncthreads();
  if (warp < 2) {
    // warp 0 finds the first tile of this block's span, warp 1 that of the next block's
    const long long total = s_total;
    const long long per = (total + gridDim.x - 1) / gridDim.x;
    long long x = per * (blockIdx.x + warp);
    PagedPlace at = {p.B, 0, 0, 0};
    if (x >= total) {
      x = total;
    } else {
      long long base = 0;
      int b = -1;
      for (int b0 = 0; b0 < p.B && b < 0; b0 += 32) {
        const long long s = b0 + lane < p.B ? (long long)s_sum[b0 + lane] * p.Hkv : 0;
        long long inc = s;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const long long o = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += o;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, base + inc > x);
        if (hit) {
          const int l = __ffs(hit) - 1;
          b = b0 + l;
          base += __shfl_sync(0xffffffffu, inc - s, l);
        } else {
          base += __shfl_sync(0xffffffffu, inc, 31);
        }
      }
      const PagedRequest r = paged_request(p, b);
      const int nt = paged_row_tiles<ROWS>(r, p.G);
      long long rem = x - base;
      const int per_head = s_sum[b];
      int h = (int)(rem / per_head);
      int k = (int)(rem - (long long)h * per_head);
      int tile = 0, n = 1;
      int run = 0;
      bool found = false;
      for (int t0 = 0; t0 < nt && !found; t0 += 32) {
        PagedUnit<ROWS, KT> u;
        u.n = 0;
        if (t0 + lane < nt) u.set(r, p.G, p.window, t0 + lane);
        int inc = u.n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += o;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, run + inc > k);
        if (hit) {
          const int l = __ffs(hit) - 1;
          tile = t0 + l;
          n = __shfl_sync(0xffffffffu, u.n, l);
          k -= run + __shfl_sync(0xffffffffu, inc - u.n, l);
          found = true;
        } else {
          run += __shfl_sync(0xffffffffu, inc, 31);
        }
      }
      if (k > 0) {
        if (k <= snap) {
          x -= k;
          k = 0;
        } else if (n - k <= snap) {                  // the next unit; its place is found by walking on
          x += n - k;
          k = 0;
          if (++tile == nt) {
            tile = 0;
            if (++h == p.Hkv) {
              h = 0;
              do { ++b; } while (b < p.B && s_sum[b] == 0);
            }
          }
        }
      }
      at = {b, h, tile, k};
    }
    if (lane == 0) {
      s_place[warp] = at;
      s_pos[warp] = x;
    }
  }
  __syncthreads();
  place = s_place[0];
  count = s_pos[1] - s_pos[0];
  __syncthreads();
}

// The unit after (b, h, tile): next row tile, next KV head, next request that has rows. False when there is none.
template <int ROWS>
__device__ __forceinline__ bool paged_next(const PagedParams& p, PagedPlace& at, PagedRequest& r) {
  at.k = 0;
  if (++at.tile < paged_row_tiles<ROWS>(r, p.G)) return true;
  at.tile = 0;
  if (++at.h < p.Hkv) return true;
  at.h = 0;
  do {
    if (++at.b >= p.B) return false;
    r = paged_request(p, at.b);
  } while (r.q == 0);
  return true;
}

// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Scores of N neighbouring keys, the first at distance d0 = (key - position), in place: raw products q.k become
// scores times log2(e). What they are made of is asked once per call, not per score.
//
// tanh(y) = 1 - 2 / (1 + e^2y): its rounding is relative to 1, which is fp32 rounding of the largest of these scores
// as long as that one is of the order of the cap. Where all 32 lanes' |y| are below 0.35, as scores far below their cap
// are, the odd Taylor polynomial up to y^9 instead (first term left out: 0.00886 y^10 of the value, 2.5e-7), which also
// leaves the exponential unit alone.
template <int N>
__device__ __forceinline__ void paged_scores(const PagedParams& p, float* x, float slope_log2, int d0) {
  if (p.cap_log2 > 0.0f) {
    const uint64_t in2 = pack2(p.cap_in, p.cap_in);
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t y = mul2(pack2(x[i], x[i + 1]), in2);
      unpack2(y, x[i], x[i + 1]);
      asm("max.f32 %0, %0, %1, %2;" : "+f"(big) : "f"(fabsf(x[i])), "f"(fabsf(x[i + 1])));
    }
    if (__any_sync(0xffffffffu, !(big < 0.35f))) {
      const uint64_t two2 = pack2(2.0f * PA_LOG2E, 2.0f * PA_LOG2E), m2 = pack2(-2.0f * p.cap_log2, -2.0f * p.cap_log2);
      const uint64_t cap2 = pack2(p.cap_log2, p.cap_log2), one2 = pack2(1.0f, 1.0f);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        float a, b;
        unpack2(mul2(pack2(x[i], x[i + 1]), two2), a, b);
        unpack2(add2(pack2(ex2(a), ex2(b)), one2), a, b);
        unpack2(fma2(pack2(rcp(a), rcp(b)), m2, cap2), x[i], x[i + 1]);
      }
    } else {
      const uint64_t cap2 = pack2(p.cap_log2, p.cap_log2);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const uint64_t y = pack2(x[i], x[i + 1]), z = mul2(y, y);
        uint64_t q = fma2(z, pack2(62.0f / 2835.0f, 62.0f / 2835.0f), pack2(-17.0f / 315.0f, -17.0f / 315.0f));
        q = fma2(z, q, pack2(2.0f / 15.0f, 2.0f / 15.0f));
        q = fma2(z, q, pack2(-1.0f / 3.0f, -1.0f / 3.0f));
        q = fma2(z, q, pack2(1.0f, 1.0f));
        unpack2(mul2(q, mul2(y, cap2)), x[i], x[i + 1]);
      }
    }
  } else {
    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
#pragma unroll
    for (int i = 0; i < N; i += 2) unpack2(mul2(pack2(x[i], x[i + 1]), scale2), x[i], x[i + 1]);
  }
  if (p.slopes) {
    const uint64_t d2 = pack2((float)d0, (float)d0);
    if (__all_sync(0xffffffffu, d0 + N <= 1)) {          // no key behind its query: |p - j| = p - j
      const uint64_t s2 = pack2(slope_log2, slope_log2);
#pragma unroll
      for (int i = 0; i < N; i += 2)
        unpack2(fma2(add2(d2, pack2((float)i, (float)(i + 1))), s2, pack2(x[i], x[i + 1])), x[i], x[i + 1]);
    } else {
      const uint64_t s2 = pack2(-slope_log2, -slope_log2);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        float a, b;
        unpack2(add2(d2, pack2((float)i, (float)(i + 1))), a, b);
        unpack2(fma2(pack2(fabsf(a), fabsf(b)), s2, pack2(x[i], x[i + 1])), x[i], x[i + 1]);
      }
    }
  }
}

template <typename T>
struct Half2Of;
template <>
struct Half2Of<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Half2Of<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// 16 bytes, or zeros when `ok` is false (nothing is read then).
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst_smem, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst_smem), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// Joins the pieces of the units that a cut divided: block (c, y) takes the unit that span c leaves unfinished,
// rows y*RB ... of its tile, one warp per row:
//     M = max m_s,  out = sum 2^(m_s - M) o_s / sum 2^(m_s - M) l_s.
constexpr int PM_WARPS = 4;
template <typename T, int D, int ROWS, int RPW>
__global__ void __launch_bounds__(PM_WARPS * 32) paged_merge_kernel(PagedParams p) {
  __shared__ float s_w[PM_WARPS][512];
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int4 d = p.ws_desc[2 * c + 1];
  if (d.x == 0) return;
  const PagedRequest r = paged_request(p, d.y);
  const int rows = min(ROWS, r.q * p.G - d.w * ROWS);
  const int row0 = (blockIdx.y * PM_WARPS + warp) * RPW;
  if (blockIdx.y * PM_WARPS * RPW >= rows) return;
  // pieces: slot 2c+1, then 2(c+1), 2(c+2), ... up to the one that ends the unit
  int last = c + 1;
  while (true) {
    const int k = last + lane;
    const int4 e = k < p.grid ? p.ws_desc[2 * k] : make_int4(0, 1, 0, 0);
    const unsigned stop = __ballot_sync(0xffffffffu, e.x == 0 || e.y != 0);
    if (stop) {
      last += __ffs(stop) - 1;
      break;
    }
    last += 32;
  }
  const int n = min(last, p.grid - 1) - c + 1;
  for (int rr = row0; rr < min(row0 + RPW, rows); ++rr) {
    float m = -INFINITY;
    for (int s = lane; s < n; s += 32) m = fmaxf(m, p.ws_ml[(int64_t)(s == 0 ? 2 * c + 1 : 2 * (c + s)) * ROWS + rr].x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ms = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    for (int s = lane; s < n; s += 32) {
      const float2 ml = p.ws_ml[(int64_t)(s == 0 ? 2 * c + 1 : 2 * (c + s)) * ROWS + rr];
      const float w = exp2f(ml.x - ms);
      s_w[warp][s] = w;
      l = fmaf(w, ml.y, l);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    __syncwarp();
    constexpr int E = D / 32;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float* o = p.ws_o + ((int64_t)(s == 0 ? 2 * c + 1 : 2 * (c + s)) * ROWS + rr) * D + lane * E;
      const float w = s_w[warp][s];
      if constexpr (E == 4) {
        const float4 v = *reinterpret_cast<const float4*>(o);
        acc[0] = fmaf(w, v.x, acc[0]); acc[1] = fmaf(w, v.y, acc[1]);
        acc[2] = fmaf(w, v.z, acc[2]); acc[3] = fmaf(w, v.w, acc[3]);
      } else {
        const float2 v = *reinterpret_cast<const float2*>(o);
        acc[0] = fmaf(w, v.x, acc[0]); acc[1] = fmaf(w, v.y, acc[1]);
      }
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);       // a NaN stays one
    const int flat = d.w * ROWS + rr, token = flat / p.G, head = d.z * p.G + (flat - token * p.G);
    const int64_t at = (int64_t)(r.first + token) * p.Hq + head;
    T* out = reinterpret_cast<T*>(p.out) + at * D + lane * E;
    if constexpr (E == 4) {
      *reinterpret_cast<uint2*>(out) = make_uint2(Half2Of<T>::pack(acc[0] * inv, acc[1] * inv), Half2Of<T>::pack(acc[2] * inv, acc[3] * inv));
    } else {
      *reinterpret_cast<uint32_t*>(out) = Half2Of<T>::pack(acc[0] * inv, acc[1] * inv);
    }
    if (p.lse && lane == 0) p.lse[at] = l == 0.0f ? -INFINITY : (ms + log2f(l)) * PA_LN2;
    __syncwarp();
  }
}

}  // namespace kvb
