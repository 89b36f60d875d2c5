// Attention of a ragged batch of new tokens over paged K/V: the kernel for few rows (decode steps, a handful of
// drafted tokens) and the entry point. Scores, visible ranges, spans and pieces: paged_common.cuh.
#include "paged_attend_tc.cu"

namespace kvb {

constexpr int PR_WARPS = 4;
constexpr int PR_THREADS = PR_WARPS * 32;
constexpr int PR_ROWS = 16;                 // rows of a unit: one mma A tile
constexpr int PR_KT = 16 * PR_WARPS;        // keys of a tile, 16 per warp
constexpr int PR_STAGES = 3;
constexpr int PR_SNAP = 1, PR_LEAST = 4;    // key tiles, see paged_common.cuh: 4096 keys x 8 heads 14.4 us, 14.9 with 2, 15.5 with 8
constexpr int PR_MAX_GRID = 296;            // two blocks per SM
constexpr float PR_LAZY = 8.0f;             // a row's reference moves when a score passes it by 2^8

template <int D>
struct RowsCfg {
  static constexpr int ROWB = D * 2;
  static constexpr int TILEB = 16 * ROWB;               // one warp's K (or V) rows of a tile
  static constexpr int STAGEB = 2 * TILEB;
  static constexpr int WARPB = PR_STAGES * STAGEB;      // also holds the warp's fp32 output tile at the end
  static constexpr int SMEM = PR_WARPS * WARPB;
  static_assert(WARPB >= PR_ROWS * D * 4, "the output tile is joined in the ring");
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// A warp streams its own 16 keys of every tile through a private ring of cp.async stages (16-byte pieces, piece c of
// row r at c ^ (r & 7): ldmatrix reads 8 rows from 8 different bank groups), so warps meet only at the end of a unit.
// Both products are mma.sync m16n8k16 with 16 rows; the score fragment is the A fragment of the second product.
// Rows of a decode step are few (q*G), so the kernel is bound by the K and V bytes, not by the tensor cores.
// Online softmax in fp32 with a reference that moves only when a score passes it by 2^8, which keeps the rescaling of
// the output out of nearly every tile; the weights are rounded to the input type for the second product, as the
// values they weigh are, and their sum is taken before that.
// Measured: 8 requests of 20001 ... 32767 tokens, 16/8 heads (813 MB) 129 us = 6.30 TB/s, 0.96 of the copy bandwidth; 16
// requests of 1000 ... 65535 tokens (1.86 GB) 275-296 us; one request of 4096 tokens 14.4 us with the join, of which 3 us
// are the span and the rest round trips to memory.
template <typename T, int D, bool MOD>
__global__ void __launch_bounds__(PR_THREADS, 2) paged_rows_kernel(PagedParams p) {
  using Cfg = RowsCfg<D>;
  constexpr int KS = D / 16;
  extern __shared__ __align__(128) uint8_t pr_smem[];
  __shared__ float2 s_ml[PR_WARPS][PR_ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  pdl_launch_dependents();

  PagedSpan span = paged_span<PR_ROWS, PR_KT, PR_THREADS>(p, reinterpret_cast<int*>(pr_smem), PR_SNAP, PR_LEAST);
  if (threadIdx.x == 0) p.ws_desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
  if (span.left <= 0) return;
  PagedPlace& at = span.at;
  PagedRequest r = paged_request(p, at.b);

  uint8_t* my = pr_smem + warp * Cfg::WARPB;
  const uint32_t my_s = smem_u32(my);
  const int pmask = (1 << p.shift) - 1;
  __syncthreads();                                       // the ring was the scheduler's scratch; descriptors cleared first

  while (true) {
    PagedUnit<PR_ROWS, PR_KT> u;
    u.set(p, r, at.tile);
    const int ntile = (int)min((long long)(u.n - at.k), span.left);
    const bool begins = at.k == 0, ends = at.k + ntile == u.n;
    const int rows = min(PR_ROWS, r.q * p.G - at.tile * PR_ROWS);
    const int key0 = (u.t0 + at.k) * PR_KT + warp * 16;
    const int32_t* table = p.table + (int64_t)at.b * p.table_st;
    const T* kbase = reinterpret_cast<const T*>(p.key) + (int64_t)at.h * p.k_sh;
    const T* vbase = reinterpret_cast<const T*>(p.value) + (int64_t)at.h * p.v_sh;

    // ---- the two rows of this lane
    uint32_t qa[KS][4];
    int lo[2], hi[2], pos[2];
    float slope[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = g + 8 * i, flat = at.tile * PR_ROWS + row;
      const bool live = row < rows;
      const int token = live ? paged_token(p, flat) : 0, head = at.h * p.G + (live ? flat - token * p.G : 0);
      const T* qr = reinterpret_cast<const T*>(p.q) + (int64_t)(r.first + token) * p.q_st + (int64_t)head * p.q_sh + 2 * t4;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qa[ks][i] = live ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks) : 0u;
        qa[ks][i + 2] = live ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 8) : 0u;
      }
      lo[i] = paged_lo(r, p.window, token);
      hi[i] = live ? paged_hi(r, token) : 0;
      pos[i] = r.kv - r.q + token;
      slope[i] = MOD && p.slopes && live ? p.slopes[head] * PA_LOG2E : 0.0f;
    }
    // keys that every row of the unit sees need no mask
    const int all_lo = paged_lo(r, p.window, paged_token(p, at.tile * PR_ROWS + rows - 1));
    const int all_hi = paged_hi(r, paged_token(p, at.tile * PR_ROWS));

    auto page_of = [&](int tile) -> int {               // lanes 16..31 mirror lanes 0..15
      const int t = key0 + tile * PR_KT + (lane & 15);
      int page = -1;
      if (tile < ntile && t >= u.lo && t < u.hi) {
        page = table[t >> p.shift];
        if (page < 0 || page >= p.num_pages) {
          atomicExch(&g_device_status, (int)KVB_BAD_ARG);
          page = -1;
        }
      }
      return page;
    };
    auto load = [&](int tile, int page) {
      constexpr int CPR = D / 8, RPI = 32 / CPR;         // pieces per row, rows per instruction
      const uint32_t sk = my_s + (tile % PR_STAGES) * Cfg::STAGEB;
      const int c = lane % CPR;
#pragma unroll
      for (int j = 0; j < 16 / RPI; ++j) {
        const int row = lane / CPR + j * RPI;
        const int pg = __shfl_sync(0xffffffffu, page, row);
        const int in = (key0 + tile * PR_KT + row) & pmask;
        const bool ok = pg >= 0;
        const uint32_t d = sk + row * Cfg::ROWB + ((c ^ (row & 7)) << 4);
        const int64_t pk = ok ? (int64_t)pg * p.k_sp + (int64_t)in * p.k_st + c * 8 : 0;
        const int64_t pv = ok ? (int64_t)pg * p.v_sp + (int64_t)in * p.v_st + c * 8 : 0;
        cp_async_16_or_zero(d, kbase + pk, ok);
        cp_async_16_or_zero(d + Cfg::TILEB, vbase + pv, ok);
      }
    };

    float o[2 * KS][4];
#pragma unroll
    for (int n = 0; n < 2 * KS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    int pg_next;
    {
      int pg[PR_STAGES];
#pragma unroll
      for (int s = 0; s < PR_STAGES; ++s) pg[s] = page_of(s);
#pragma unroll
      for (int s = 0; s < PR_STAGES - 1; ++s) {
        if (s < ntile) load(s, pg[s]);
        cp_async_commit();
      }
      pg_next = pg[PR_STAGES - 1];
    }

    for (int i = 0; i < ntile; ++i) {
      const int pg_after = page_of(i + PR_STAGES);
      if (i + PR_STAGES - 1 < ntile) load(i + PR_STAGES - 1, pg_next);
      cp_async_commit();
      pg_next = pg_after;
      cp_async_wait<PR_STAGES - 1>();
      __syncwarp();

      const uint32_t sk = my_s + (i % PR_STAGES) * Cfg::STAGEB, sv = sk + Cfg::TILEB;
      const int t0 = key0 + i * PR_KT;
      float c[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // matrices: keys 0-7 | 0-7 | 8-15 | 8-15 of the tile, d pieces 2ks | 2ks+1 | 2ks | 2ks+1
        const int row = (lane & 7) + ((lane >> 4) << 3), piece = 2 * ks + ((lane >> 3) & 1);
        uint32_t kb[4];
        ldsm_x4(kb, sk + row * Cfg::ROWB + ((piece ^ (row & 7)) << 4));
        Half2Of<T>::mma(c[0], qa[ks], kb[0], kb[1]);
        Half2Of<T>::mma(c[1], qa[ks], kb[2], kb[3]);
      }
      // ---- scores times log2(e); element e of tile n: row g + 8*(e/2), key t0 + 8n + 2*t4 + e%2
      const bool edge = t0 < all_lo || t0 + 16 > all_hi;
      float x[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] = MOD ? c[n][e] : c[n][e] * p.scale_log2;
      if constexpr (MOD) {
        paged_scale<8>(p, &x[0][0]);
        if (p.slopes) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[n][e] = fmaf(-slope[e >> 1], fabsf((float)(t0 + 8 * n + 2 * t4 + (e & 1) - pos[e >> 1])), x[n][e]);
        }
      }
      if (edge)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = t0 + 8 * n + 2 * t4 + (e & 1), w = e >> 1;
            if (t < lo[w] || t >= hi[w]) x[n][e] = -INFINITY;
          }
      float mx[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        mx[w] = fmaxf(fmaxf(x[0][2 * w], x[0][2 * w + 1]), fmaxf(x[1][2 * w], x[1][2 * w + 1]));
        mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 1));
        mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 2));
      }
      const bool move0 = mx[0] > m[0] + PR_LAZY, move1 = mx[1] > m[1] + PR_LAZY;
      if (__any_sync(0xffffffffu, move0 || move1)) {
        float a[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const bool mv = w == 0 ? move0 : move1;
          const float mn = mv ? mx[w] : m[w];
          a[w] = mv ? exp2f(m[w] - mn) : 1.0f;
          m[w] = mn;
          l[w] *= a[w];
        }
#pragma unroll
        for (int n = 0; n < 2 * KS; ++n) {
          o[n][0] *= a[0]; o[n][1] *= a[0];
          o[n][2] *= a[1]; o[n][3] *= a[1];
        }
      }
      const float ms[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[n][e] = ex2(x[n][e] - ms[e >> 1]);
          l[e >> 1] += x[n][e];
        }
      constexpr float W = Half2Of<T>::WEIGHT;
      uint32_t pa[4];
      pa[0] = Half2Of<T>::pack(W * x[0][0], W * x[0][1]);
      pa[1] = Half2Of<T>::pack(W * x[0][2], W * x[0][3]);
      pa[2] = Half2Of<T>::pack(W * x[1][0], W * x[1][1]);
      pa[3] = Half2Of<T>::pack(W * x[1][2], W * x[1][3]);
#pragma unroll
      for (int n = 0; n < KS; ++n) {
        // matrices: keys 0-7 | 8-15 | 0-7 | 8-15, d pieces 2n | 2n | 2n+1 | 2n+1
        const int row = lane & 15, piece = 2 * n + (lane >> 4);
        uint32_t vb[4];
        ldsm_x4_t(vb, sv + row * Cfg::ROWB + ((piece ^ (row & 7)) << 4));
        Half2Of<T>::mma(o[2 * n], pa, vb[0], vb[1]);
        Half2Of<T>::mma(o[2 * n + 1], pa, vb[2], vb[3]);
      }
      __syncwarp();                                      // every lane has read the stage that is loaded next
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- join the warps' outputs in the ring (each in its own part), then write the unit or its piece
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
      if (t4 == 0) s_ml[warp][g + 8 * w] = make_float2(m[w], l[w]);
    }
    float* so = reinterpret_cast<float*>(my);
#pragma unroll
    for (int n = 0; n < 2 * KS; ++n) {
      *reinterpret_cast<float2*>(so + g * D + 8 * n + 2 * t4) = make_float2(o[n][0], o[n][1]);
      *reinterpret_cast<float2*>(so + (g + 8) * D + 8 * n + 2 * t4) = make_float2(o[n][2], o[n][3]);
    }
    __syncthreads();
    constexpr int E = D / 32;
    const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
    for (int row = warp; row < rows; row += PR_WARPS) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < PR_WARPS; ++w) M = fmaxf(M, s_ml[w][row].x);
      const float ms = M == -INFINITY ? 0.0f : M;
      float L = 0.0f, acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll
      for (int w = 0; w < PR_WARPS; ++w) {
        const float2 ml = s_ml[w][row];
        float f = exp2f(ml.x - ms);
        L = fmaf(f, ml.y, L);
        f *= 1.0f / Half2Of<T>::WEIGHT;
        const float* src = reinterpret_cast<const float*>(pr_smem + w * Cfg::WARPB) + row * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(f, src[e], acc[e]);
      }
      if (begins && ends) {
        const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);
        const int flat = at.tile * PR_ROWS + row, token = paged_token(p, flat), head = at.h * p.G + (flat - token * p.G);
        const int64_t to = (int64_t)(r.first + token) * p.Hq + head;
        uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + to * D + lane * E);
#pragma unroll
        for (int e = 0; e < E; e += 2) out[e / 2] = Half2Of<T>::pack(acc[e] * inv, acc[e + 1] * inv);
        if (p.lse && lane == 0) p.lse[to] = L == 0.0f ? -INFINITY : (ms + log2f(L)) * PA_LN2;
      } else {
        float* dst = p.ws_o + ((int64_t)slot * PR_ROWS + row) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = acc[e];
        if (lane == 0) p.ws_ml[(int64_t)slot * PR_ROWS + row] = make_float2(M, L);
      }
    }
    if (begins && !ends && threadIdx.x == 0) {
      p.ws_desc[2 * blockIdx.x] = make_int4(paged_pieces(span.per, span.x, u.n, PR_SNAP, blockIdx.x), at.h, at.tile, 0);
      p.ws_desc[2 * blockIdx.x + 1] = make_int4(r.first, r.q, 0, 0);
    }
    span.left -= ntile;
    span.x += ntile;
    if (span.left <= 0 || !paged_next<PR_ROWS>(p, at, r)) break;
    __syncthreads();                                     // the ring is read no more
  }
}

static inline int64_t paged_tile_bound(int64_t N, int B, int Hkv, int G, int64_t keys, int rows, int kt) {
  const int64_t units = ((N * G + rows - 1) / rows + B) * Hkv;
  return units * ((keys + kt - 1) / kt + 1);
}
// Few rows per request: the kernel bound by K and V bytes. More: the tensor-core kernel. Either takes any shape.
static inline bool paged_few_rows(int N, int B, int G, int max_q) {
  return (int64_t)(max_q > 0 ? max_q : N == B ? 1 : N) * G <= PR_ROWS;
}
struct PagedSizes { bool few; int grid, rows, few_tiles; };
static inline PagedSizes paged_sizes(int N, int B, int Hkv, int G, int64_t keys, int max_q) {
  PagedSizes s;
  s.few = paged_few_rows(N, B, G, max_q);
  s.rows = s.few ? PR_ROWS : PT_ROWS;
  const int64_t most = s.few ? PR_MAX_GRID : PT_MAX_GRID;
  const int64_t t = paged_tile_bound(N, B, Hkv, G, keys, s.rows, s.few ? PR_KT : PT_KT);
  s.grid = (int)(t < most ? t : most);
  s.few_tiles = t < 0x7fffffff;
  return s;
}
static inline size_t paged_ws_bytes(int grid, int rows, int D) {
  return round_up((size_t)2 * grid * rows * D * 4, 256) + round_up((size_t)2 * grid * rows * 8, 256) + (size_t)2 * grid * 16;
}

template <typename T, int D, bool MOD>
static int launch_paged_rows(PagedParams& p, int device, cudaStream_t st) {
  static std::atomic<bool> done[KVB_MAX_DEVICES];
  const int rc = ensure_dynamic_smem(paged_rows_kernel<T, D, MOD>, done, device, RowsCfg<D>::SMEM);
  if (rc != KVB_OK) return rc;
  const size_t sched = (size_t)p.B * 4;
  const size_t smem = sched > RowsCfg<D>::SMEM ? sched : RowsCfg<D>::SMEM;
  static_assert(PA_MAX_B * 4 <= RowsCfg<D>::SMEM, "the scheduler's scratch is the ring");
  KVB_CHECK_CUDA(launch_kernel(paged_rows_kernel<T, D, MOD>, dim3(p.grid), dim3(PR_THREADS), smem, st, p));
  if (p.grid > 1) {
    ChainLaunchScope chain;
    chain.on();
    KVB_CHECK_CUDA(launch_kernel(paged_merge_kernel<T, D, PR_ROWS, 1>, dim3(p.grid, PR_ROWS / PM_WARPS),
                                 dim3(PM_WARPS * 32), 0, st, p));
  }
  return KVB_OK;
}

// A tensor of `rank` dimensions (the first contiguous) in boxes of 64 elements, 128-byte swizzle: the layout the tensor
// core reads. False when the driver takes no such map (a stride of 0 or beyond its range); rows are copied one by one then.
template <typename T>
static bool paged_tensor_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const int64_t* strides,
                             const cuuint32_t* box) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess) fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!encode) return false;
  cuuint64_t bytes[3];
  for (int i = 0; i + 1 < rank; ++i) {
    const int64_t s = dims[i + 1] > 1 ? strides[i] : (int64_t)dims[0];      // a dimension of one element has no stride of its own
    if (s < (int64_t)dims[0]) return false;
    bytes[i] = (cuuint64_t)s * 2;
  }
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return encode(map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                (cuuint32_t)rank, const_cast<void*>(base), dims, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool MOD>
static int launch_paged_chunk(PagedParams& p, int device, cudaStream_t st) {
  static std::atomic<bool> done[KVB_MAX_DEVICES];
  const int rc = ensure_dynamic_smem(paged_chunk_kernel<T, D, MOD>, done, device, PtCfg<D>::SMEM);
  if (rc != KVB_OK) return rc;
  static_assert(PA_MAX_B * 4 <= PtCfg<D>::OFF_BAR - PtCfg<D>::OFF_KV, "the scheduler's scratch is the ring");
  CUtensorMap kmap = {}, vmap = {}, qmap = {};
  const int P = 1 << p.shift, box = P < PT_KT ? P : PT_KT;
  const cuuint64_t pool[4] = {(cuuint64_t)D, (cuuint64_t)P, (cuuint64_t)p.Hkv, (cuuint64_t)p.num_pages};
  const int64_t ks[3] = {p.k_st, p.k_sh, p.k_sp}, vs[3] = {p.v_st, p.v_sh, p.v_sp};
  const cuuint32_t rows[4] = {64, (cuuint32_t)box, 1, 1};
  p.box = P >= 8 && paged_tensor_map<T>(&kmap, p.key, 4, pool, ks, rows) && paged_tensor_map<T>(&vmap, p.value, 4, pool, vs, rows) ? box : 0;
  const cuuint64_t query[3] = {(cuuint64_t)D, (cuuint64_t)p.Hq, (cuuint64_t)p.N};
  const int64_t qs[2] = {p.q_sh, p.q_st};
  const cuuint32_t tokens[3] = {64, (cuuint32_t)p.G, (cuuint32_t)(128 / p.G)};
  p.qbox = p.G <= 128 && 128 % p.G == 0 && paged_tensor_map<T>(&qmap, p.q, 3, query, qs, tokens) ? 128 / p.G : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid);
  cfg.blockDim = dim3(PT_THREADS);
  cfg.dynamicSmemBytes = PtCfg<D>::SMEM;
  cfg.stream = st;
  KVB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_chunk_kernel<T, D, MOD>, p, kmap, vmap, qmap));
  if (p.grid > 1) {
    ChainLaunchScope chain;
    chain.on();
    KVB_CHECK_CUDA(launch_kernel(paged_merge_kernel<T, D, PT_ROWS, 4>, dim3(p.grid, PT_ROWS / (4 * PM_WARPS)),
                                 dim3(PM_WARPS * 32), 0, st, p));
  }
  return KVB_OK;
}

template <typename T, int D>
static int launch_paged(PagedParams& p, bool few, bool mod, int device, cudaStream_t st) {
  if (!few) return mod ? launch_paged_chunk<T, D, true>(p, device, st) : launch_paged_chunk<T, D, false>(p, device, st);
  return mod ? launch_paged_rows<T, D, true>(p, device, st) : launch_paged_rows<T, D, false>(p, device, st);
}

static int paged_shape(const kvb_paged_attend_params* p, int64_t& keys) {
  if (p->N < 0 || p->B < 1 || p->B > PA_MAX_B || p->Hkv < 1 || p->Hq < 1 || p->Hq % p->Hkv || p->W < 1 || p->num_pages < 1)
    return KVB_BAD_SHAPE;
  if (p->D != 64 && p->D != 128) return KVB_BAD_SHAPE;
  if (!page_tokens_ok(p->page_tokens)) return KVB_BAD_SHAPE;
  keys = (int64_t)p->W * p->page_tokens;
  if (keys > 0x40000000) return KVB_BAD_SHAPE;
  // rows, and key tiles of one KV head of one request, are counted in 32 bits
  const int64_t G = p->Hq / p->Hkv;
  if (p->N * G > 0x3fffffff || (p->N * G / PR_ROWS + 1) * (keys / PR_KT + 2) > 0x7fffffff) return KVB_BAD_SHAPE;
  return KVB_OK;
}

}  // namespace kvb

extern "C" __attribute__((visibility("default"))) size_t kvb_paged_attend_workspace_bytes(
    int N, int B, int Hq, int Hkv, int W, int page_tokens, int D, int max_q) {
  using namespace kvb;
  kvb_paged_attend_params q = {};
  q.N = N; q.B = B; q.Hq = Hq; q.Hkv = Hkv; q.W = W; q.page_tokens = page_tokens; q.D = D; q.num_pages = 1;
  int64_t keys;
  if (paged_shape(&q, keys) != KVB_OK) return 0;
  const PagedSizes s = paged_sizes(N, B, Hkv, Hq / Hkv, keys, max_q);
  return paged_ws_bytes(s.grid, s.rows, D);
}

extern "C" __attribute__((visibility("default"))) int kvb_paged_attend(const kvb_paged_attend_params* a, int device,
                                                                       void* stream) {
  using namespace kvb;
  if (!a || !a->query || !a->key_pool || !a->value_pool || !a->page_table || !a->kv_len || !a->out || !a->workspace)
    return KVB_BAD_ARG;
  int64_t keys;
  const int rc = paged_shape(a, keys);
  if (rc != KVB_OK) return rc;
  if (a->max_q < 0) return KVB_BAD_ARG;
  if (a->page_table_stride < a->W || (a->cu_q == nullptr && a->N != a->B)) return KVB_BAD_SHAPE;
  if (a->elem_type != 0 && a->elem_type != 1) return KVB_BAD_ARG;
  if (!(a->scaling > 0.0f) || a->scaling > 3.0e38f || !(a->softcap >= 0.0f) || a->softcap > 3.0e38f || a->window < 0 ||
      (a->softcap > 0.0f && !(a->scaling / a->softcap < 3.0e38f)))
    return KVB_BAD_ARG;
  const int64_t strides[] = {a->q_st, a->q_sh, a->k_sp, a->k_sh, a->k_st, a->v_sp, a->v_sh, a->v_st};
  for (int64_t s : strides)
    if (s % 8 || s < 0) return KVB_BAD_ALIGN;
  if (!aligned_to(a->query, 16) || !aligned_to(a->key_pool, 16) || !aligned_to(a->value_pool, 16) ||
      !aligned_to(a->out, 16) || !aligned_to(a->workspace, 256))
    return KVB_BAD_ALIGN;
  DeviceGuard guard(device);
  if (!guard.ok) return KVB_BAD_DEVICE;
  if (a->N == 0) return KVB_OK;
  PagedParams p = {};
  p.q = a->query; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.key = a->key_pool; p.k_sp = a->k_sp; p.k_sh = a->k_sh; p.k_st = a->k_st;
  p.value = a->value_pool; p.v_sp = a->v_sp; p.v_sh = a->v_sh; p.v_st = a->v_st;
  p.table = a->page_table; p.table_st = a->page_table_stride; p.W = a->W; p.shift = log2_int(a->page_tokens);
  p.num_pages = a->num_pages;
  p.cu_q = a->cu_q; p.kv_len = a->kv_len; p.prefix = a->prefix_len; p.slopes = a->slopes;
  p.N = a->N; p.B = a->B; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv; p.window = a->window;
  p.g_shift = (p.G & (p.G - 1)) == 0 ? log2_int(p.G) : -1;
  p.scale_log2 = a->scaling * PA_LOG2E;
  if (a->softcap > 0.0f) { p.cap_in = a->scaling / a->softcap; p.cap_log2 = a->softcap * PA_LOG2E; }
  p.out = a->out; p.lse = a->lse;
  const PagedSizes s = paged_sizes(a->N, a->B, a->Hkv, p.G, keys, a->max_q);
  p.grid = s.grid;
  p.few_tiles = s.few_tiles;
  if (a->workspace_bytes < paged_ws_bytes(s.grid, s.rows, a->D)) return KVB_WORKSPACE_TOO_SMALL;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.ws_o = reinterpret_cast<float*>(ws);
  ws += round_up((size_t)2 * s.grid * s.rows * a->D * 4, 256);
  p.ws_ml = reinterpret_cast<float2*>(ws);
  ws += round_up((size_t)2 * s.grid * s.rows * 8, 256);
  p.ws_desc = reinterpret_cast<int4*>(ws);
  const bool mod = a->softcap > 0.0f || a->slopes != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->elem_type == 0)
    return a->D == 128 ? launch_paged<__nv_bfloat16, 128>(p, s.few, mod, device, st) : launch_paged<__nv_bfloat16, 64>(p, s.few, mod, device, st);
  return a->D == 128 ? launch_paged<__half, 128>(p, s.few, mod, device, st) : launch_paged<__half, 64>(p, s.few, mod, device, st);
}
