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
  int g_shift;                                       // log2(G), -1 when it is not a power of two
  float scale_log2;                                  // scaling * log2(e)
  float cap_in, cap_log2;                            // scaling / softcap, softcap * log2(e); cap_log2 == 0: none
  void* out;                                         // [N,Hq,D]
  float* lse;                                        // [N,Hq] or NULL
  float* ws_o;                                       // [2*grid][ROWS][D] un-normalised outputs of unit pieces
  float2* ws_ml;                                     // [2*grid][ROWS] (m, l)
  int4* ws_desc;                                     // [2*grid]: see PieceDesc
  int grid;
  int few_tiles;                                     // whether all key tiles can be counted in 31 bits
  int box;                                           // rows per TMA box of a pool, 0: no TMA
  int qbox;                                          // tokens per TMA box of the query, 0: no TMA
};

// ws_desc[2c], ws_desc[2c+1]: the unit that span c begins and a later one ends: {pieces, KV head, row tile, 0} and the
// request's {first row, new tokens, 0, 0}; pieces == 0 when there is none. The first piece lies at slot 2c+1, the
// pieces of the spans after it at slots 2(c+1), 2(c+2), ...

// Row n of a request belongs to token n / G.
__device__ __forceinline__ int paged_token(const PagedParams& p, int n) { return p.g_shift >= 0 ? n >> p.g_shift : n / p.G; }

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
  const int most = p.W << p.shift;                     // at most 2^30
  r.kv = max(p.kv_len[b], 0);
  if (r.kv > most) {
    r.kv = most;
    atomicExch(&g_device_status, (int)KVB_BAD_ARG);
  }
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
  __device__ __forceinline__ void set(const PagedParams& p, const PagedRequest& r, int tile) {
    const int i0 = paged_token(p, tile * ROWS), i1 = min(r.q - 1, paged_token(p, tile * ROWS + ROWS - 1));
    lo = paged_lo(r, p.window, i0);
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
struct PagedSpan {
  PagedPlace at;                                       // the block's first key tile, at position x of all
  long long x, left, per;                              // how many it has; the length of a span before its ends are moved
};

__device__ __forceinline__ long long paged_div(long long a, long long b) {
  return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);      // a 64-bit division takes a hundred instructions
}

// Key tiles of one KV head of the request of every lane (all lanes call).
template <int ROWS, int KT>
__device__ __forceinline__ int paged_lane_sum(const PagedParams& p, const PagedRequest& r, int lane) {
  const int tiles = paged_row_tiles<ROWS>(r, p.G);
  int sum = 0;
  if (tiles <= 4)
    for (int t = 0; t < tiles; ++t) {
      PagedUnit<ROWS, KT> u;
      u.set(p, r, t);
      sum += u.n;
    }
  unsigned big = __ballot_sync(0xffffffffu, tiles > 4);
  while (big) {
    const int src = __ffs(big) - 1;
    big &= big - 1;
    const PagedRequest rr = {0, __shfl_sync(0xffffffffu, r.q, src), __shfl_sync(0xffffffffu, r.kv, src), __shfl_sync(0xffffffffu, r.pre, src)};
    const int nt = __shfl_sync(0xffffffffu, tiles, src);
    int part = 0;
    for (int t = lane; t < nt; t += 32) {
      PagedUnit<ROWS, KT> u;
      u.set(p, rr, t);
      part += u.n;
    }
    part = __reduce_add_sync(0xffffffffu, part);
    if (lane == src) sum = part;
  }
  return sum;
}

// The row tile of a request in which key tile k of one KV head lies; k becomes its place in the unit, n the unit's length.
template <int ROWS, int KT>
__device__ __forceinline__ int paged_find_tile(const PagedParams& p, const PagedRequest& r, int nt, int& k, int& n, int lane) {
  int run = 0;
  for (int t0 = 0; t0 < nt; t0 += 32) {
    PagedUnit<ROWS, KT> u;
    u.n = 0;
    if (t0 + lane < nt) u.set(p, r, t0 + lane);
    int inc = u.n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run + inc > k);
    if (hit) {
      const int l = __ffs(hit) - 1;
      n = __shfl_sync(0xffffffffu, u.n, l);
      k -= run + __shfl_sync(0xffffffffu, inc - u.n, l);
      return t0 + l;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  return nt;
}

// Moves a cut (at.k key tiles into a unit of n, position x) to the unit's edge when it lies within `snap` of one. True
// when that is the end of the request's last unit: the place is then the next request that has rows.
template <typename I>
__device__ __forceinline__ bool paged_snap(const PagedParams& p, PagedPlace& at, I& x, int n, int nt, int snap) {
  if (at.k == 0) return false;
  if (at.k <= snap) {
    x -= at.k;
    at.k = 0;
  } else if (n - at.k <= snap) {
    x += n - at.k;
    at.k = 0;
    if (++at.tile == nt) {
      at.tile = 0;
      if (++at.h == p.Hkv) {
        at.h = 0;
        return true;
      }
    }
  }
  return false;
}

// Cuts the work. Called by every thread of the block; s_sum: B words of shared memory, free again afterwards. With up
// to 32 requests every warp finds the span by itself, one request per lane, after one round trip to memory and with
// little code: what a block does before its first load costs a short call more than all the rest (this part took 9500
// cycles when one routine served all cases).
template <int ROWS, int KT, int THREADS>
__device__ __forceinline__ PagedSpan paged_span(const PagedParams& p, int* s_sum, int snap, int least) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  PagedSpan out;
  out.at = {p.B, 0, 0, 0};
  if (p.B <= 32 && p.few_tiles) {
    PagedRequest mine = {0, 0, 0, 0};
    if (lane < p.B) mine = paged_request(p, lane);
    const int tiles = paged_row_tiles<ROWS>(mine, p.G);
    int sum;
    if (__any_sync(0xffffffffu, tiles > 1)) {
      sum = paged_lane_sum<ROWS, KT>(p, mine, lane);
    } else {
      PagedUnit<ROWS, KT> u;
      u.set(p, mine, 0);
      sum = tiles > 0 ? u.n : 0;
    }
    int inc = sum * p.Hkv;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    const int total = __shfl_sync(0xffffffffu, inc, 31);
    const int per = max(least, (int)(((unsigned)total + gridDim.x - 1) / gridDim.x));
    int x = 0, end = 0;
#pragma unroll 1
    for (int i = 1; i >= 0; --i) {                       // the end, then the beginning
      const long long want = (long long)per * (blockIdx.x + i);
      x = want < total ? (int)want : total;
      if (x < total) {
        const int b = __ffs(__ballot_sync(0xffffffffu, inc > x)) - 1;
        const int per_head = __shfl_sync(0xffffffffu, sum, b), rem = x - __shfl_sync(0xffffffffu, inc - sum * p.Hkv, b);
        const int nt = __shfl_sync(0xffffffffu, tiles, b);
        int n = per_head;
        out.at = {b, rem / per_head, 0, rem % per_head};
        if (nt > 1) {
          const PagedRequest r = {0, __shfl_sync(0xffffffffu, mine.q, b), __shfl_sync(0xffffffffu, mine.kv, b), __shfl_sync(0xffffffffu, mine.pre, b)};
          out.at.tile = paged_find_tile<ROWS, KT>(p, r, nt, out.at.k, n, lane);
        }
        if (paged_snap(p, out.at, x, n, nt, snap)) {
          const unsigned rows = __ballot_sync(0xffffffffu, sum > 0) & (0xfffffffeu << b);
          out.at.b = rows ? __ffs(rows) - 1 : p.B;
        }
      }
      if (i == 1) end = x;
    }
    out.x = x;
    out.left = end - x;
    out.per = per;
    return out;
  }
  __shared__ long long s_total;
  __shared__ PagedPlace s_place;
  __shared__ long long s_pos[2];
  for (int b0 = warp * 32; b0 < p.B; b0 += THREADS) {
    PagedRequest r = {0, 0, 0, 0};
    if (b0 + lane < p.B) r = paged_request(p, b0 + lane);
    const int sum = paged_lane_sum<ROWS, KT>(p, r, lane);
    if (b0 + lane < p.B) s_sum[b0 + lane] = sum;
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
  const long long total = s_total;
  out.per = max((long long)least, paged_div(total + gridDim.x - 1, gridDim.x));
  if (warp < 2) {
    // warp 0 finds the first tile of this block's span, warp 1 that of the next block's
    long long x = min(total, out.per * (blockIdx.x + warp));
    PagedPlace at = {p.B, 0, 0, 0};
    if (x < total) {
      long long base = 0;
      int b = -1;
      for (int b0 = 0; b < 0; b0 += 32) {
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
      const int nt = paged_row_tiles<ROWS>(r, p.G), per_head = s_sum[b];
      const long long rem = x - base;
      at = {b, (int)paged_div(rem, per_head), 0, 0};
      at.k = (int)(rem - (long long)at.h * per_head);
      int n = per_head;
      at.tile = paged_find_tile<ROWS, KT>(p, r, nt, at.k, n, lane);
      if (paged_snap(p, at, x, n, nt, snap))
        do { ++at.b; } while (at.b < p.B && s_sum[at.b] == 0);
    }
    if (lane == 0) {
      if (warp == 0) s_place = at;
      s_pos[warp] = x;
    }
  }
  __syncthreads();
  out.at = s_place;
  out.x = s_pos[0];
  out.left = s_pos[1] - s_pos[0];
  __syncthreads();
  return out;
}

// How many pieces the unit [x - k, x - k + n) has whose first piece span c holds, when span c ends before the unit does:
// the cuts behind c that fall inside it, none within `snap` of its edges.
__device__ __forceinline__ int paged_pieces(long long per, long long begin, int n, int snap, int c) {
  return (int)(paged_div(begin + n - snap - 1, per) - c) + 1;
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

// N raw products q.k of one or more rows become scores times log2(e), in place; all lanes call. What they are made of
// is asked once per call, not per score.
//
// tanh(y) = 1 - 2 / (1 + e^2y): its rounding is relative to 1, which is fp32 rounding of the largest of these scores
// as long as that one is of the order of the cap. Where all 32 lanes' |y| are below 0.35, as scores far below their cap
// are, the odd Taylor polynomial up to y^9 instead (first term left out: 0.00886 y^10 of the value, 2.5e-7), which also
// leaves the exponential unit alone.
template <int N>
__device__ __forceinline__ void paged_scale(const PagedParams& p, float* x) {
  if (p.cap_log2 > 0.0f) {
    const uint64_t in2 = pack2(p.cap_in, p.cap_in);
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      unpack2(mul2(pack2(x[i], x[i + 1]), in2), x[i], x[i + 1]);
      asm("max.f32 %0, %0, %1, %2;" : "+f"(big) : "f"(fabsf(x[i])), "f"(fabsf(x[i + 1])));
    }
    const uint64_t cap2 = pack2(p.cap_log2, p.cap_log2);
    if (__any_sync(0xffffffffu, !(big < 0.35f))) {
      const uint64_t two2 = pack2(2.0f * PA_LOG2E, 2.0f * PA_LOG2E), m2 = pack2(-2.0f * p.cap_log2, -2.0f * p.cap_log2);
      const uint64_t one2 = pack2(1.0f, 1.0f);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        float a, b;
        unpack2(mul2(pack2(x[i], x[i + 1]), two2), a, b);
        unpack2(add2(pack2(ex2(a), ex2(b)), one2), a, b);
        unpack2(fma2(pack2(rcp(a), rcp(b)), m2, cap2), x[i], x[i + 1]);
      }
    } else {
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
}
// The distance term of N neighbouring keys, the first at distance d0 = key - position. Distances are whole numbers, exact in
// fp32 up to 2^24: four running pairs instead of a constant for each.
template <int N>
__device__ __forceinline__ void paged_bias(float* x, float slope_log2, int d0) {
  constexpr int R = N >= 8 ? 4 : N / 2;
  const bool behind = __any_sync(0xffffffffu, d0 + N > 1);       // some key behind its query: |p - j| is not p - j
  const float s = behind ? -slope_log2 : slope_log2;
  const uint64_t s2 = pack2(s, s), step = pack2((float)(2 * R), (float)(2 * R));
  const float f0 = (float)d0;
  uint64_t d[R];
#pragma unroll
  for (int i = 0; i < R; ++i) d[i] = pack2(f0 + (float)(2 * i), f0 + (float)(2 * i + 1));
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float a, b;
    unpack2(d[i % R], a, b);
    if (behind) { a = fabsf(a); b = fabsf(b); }
    unpack2(fma2(pack2(a, b), s2, pack2(x[2 * i], x[2 * i + 1])), x[2 * i], x[2 * i + 1]);
    if (i + R < N / 2) d[i % R] = add2(d[i % R], step);
  }
}
// Bit i: whether key t + i lies in [lo, hi), for 32 keys.
__device__ __forceinline__ uint32_t paged_seen(int t, int lo, int hi) {
  const int a = min(max(lo - t, 0), 32), b = min(max(hi - t, 0), 32);
  const uint32_t below = a < 32 ? (1u << a) - 1u : 0xffffffffu, upto = b < 32 ? (1u << b) - 1u : 0xffffffffu;
  return upto & ~below;
}

// WEIGHT: what the weights of the second product are multiplied by before they are rounded. A fresh weight is at most 1, a
// stale one 2^8; times 2^7 they reach 2^15, inside fp16's range, and small ones keep its normal bits down to 2^-21. bf16
// needs none. The sum of weights is taken without it (a row with one key then has the sum 1 and an exact logarithm).
template <typename T>
struct Half2Of;
template <>
struct Half2Of<__nv_bfloat16> {
  static constexpr float WEIGHT = 1.0f;
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
  static constexpr float WEIGHT = 128.0f;
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
// Bound by round trips to L2: the descriptor, then (m, l) of up to 32 pieces at once and the outputs of 16 (rows x pieces)
// at a time; 3-10 us.
constexpr int PM_WARPS = 4;
template <typename T, int D, int ROWS, int RPW>
__global__ void __launch_bounds__(PM_WARPS * 32) paged_merge_kernel(PagedParams p) {
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int4 d = p.ws_desc[2 * c], e = p.ws_desc[2 * c + 1];
  const int n = d.x;
  if (n == 0) return;
  const int rows = min(ROWS, e.y * p.G - d.z * ROWS);
  const int row0 = (blockIdx.y * PM_WARPS + warp) * RPW;
  if (row0 >= rows) return;
  constexpr int E = D / 32;
  auto slot = [&](int s) -> int64_t { return s == 0 ? 2 * c + 1 : 2 * (c + s); };
  // the warp's rows side by side, so that a round trip serves all of them
  float m[RPW], l[RPW], acc[RPW][E];
#pragma unroll
  for (int q = 0; q < RPW; ++q) {
    m[q] = -INFINITY;
    l[q] = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[q][i] = 0.0f;
  }
  for (int s0 = 0; s0 < n; s0 += 32) {
    float2 ml[RPW];
    float w[RPW];
#pragma unroll
    for (int q = 0; q < RPW; ++q)
      ml[q] = s0 + lane < n && row0 + q < rows ? p.ws_ml[slot(s0 + lane) * ROWS + row0 + q] : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int q = 0; q < RPW; ++q) {
      float top = ml[q].x;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m[q], top), ms = mn == -INFINITY ? 0.0f : mn;
      const float old = exp2f(m[q] - ms);
      w[q] = exp2f(ml[q].x - ms);
      float part = w[q] * ml[q].y;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      l[q] = fmaf(l[q], old, part);
      m[q] = mn;
#pragma unroll
      for (int i = 0; i < E; ++i) acc[q][i] *= old;
    }
    const int k = min(32, n - s0);
    constexpr int U = 16 / RPW;
#pragma unroll 1
    for (int s1 = 0; s1 < k; s1 += U) {
      float v[U][RPW][E];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int q = 0; q < RPW; ++q) {
          const bool have = s1 + u < k && row0 + q < rows;
          const float* o = p.ws_o + (slot(s0 + s1 + u) * ROWS + row0 + q) * D + lane * E;
          if constexpr (E == 4) {
            const float4 t = have ? *reinterpret_cast<const float4*>(o) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v[u][q][0] = t.x; v[u][q][1] = t.y; v[u][q][2] = t.z; v[u][q][3] = t.w;
          } else {
            const float2 t = have ? *reinterpret_cast<const float2*>(o) : make_float2(0.0f, 0.0f);
            v[u][q][0] = t.x; v[u][q][1] = t.y;
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int q = 0; q < RPW; ++q) {
          const float f = __shfl_sync(0xffffffffu, w[q], (s1 + u) & 31);
          if (s1 + u < k)
#pragma unroll
            for (int i = 0; i < E; ++i) acc[q][i] = fmaf(f, v[u][q][i], acc[q][i]);
        }
    }
  }
#pragma unroll
  for (int q = 0; q < RPW; ++q) {
    if (row0 + q >= rows) break;
    const float inv = l[q] > 0.0f ? 1.0f / l[q] : (l[q] == 0.0f ? 0.0f : l[q]);       // a NaN stays one
    const int flat = d.z * ROWS + row0 + q, token = paged_token(p, flat), head = d.y * p.G + (flat - token * p.G);
    const int64_t at = (int64_t)(e.x + token) * p.Hq + head;
    T* out = reinterpret_cast<T*>(p.out) + at * D + lane * E;
    if constexpr (E == 4) {
      *reinterpret_cast<uint2*>(out) = make_uint2(Half2Of<T>::pack(acc[q][0] * inv, acc[q][1] * inv), Half2Of<T>::pack(acc[q][2] * inv, acc[q][3] * inv));
    } else {
      *reinterpret_cast<uint32_t*>(out) = Half2Of<T>::pack(acc[q][0] * inv, acc[q][1] * inv);
    }
    if (p.lse && lane == 0) p.lse[at] = l[q] == 0.0f ? -INFINITY : ((m[q] == -INFINITY ? 0.0f : m[q]) + log2f(l[q])) * PA_LN2;
  }
}

}  // namespace kvb
