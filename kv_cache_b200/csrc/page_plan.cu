// Bookkeeping of a ragged batch over paged K/V, on the device: which page and row every new token gets
// (page_plan_kernel), and the store of the new K and V rows there (paged_append_kernel).
#include "common.cuh"

namespace kvb {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_MAX_CTAS = 8;                   // one portable cluster
constexpr int PLAN_MAX_B = 8192;

struct PagePlanParams {
  const int32_t* kv_len; const int32_t* q_len; const uint8_t* finished; int B;
  int32_t* table; int64_t table_st; int W;
  int32_t* free_pages; int num_pages; const int32_t* free_count;
  int shift; int capacity;
  int32_t* cu_q; int32_t* kv_len_out; int32_t* free_count_out;
  int64_t* slot; int32_t* position; int32_t* request; int32_t* status;
};

struct PlanSums { long long q, take, gone; };

__device__ __forceinline__ PlanSums plan_shfl_up(const PlanSums& a, int d) {
  return {__shfl_up_sync(0xffffffffu, a.q, d), __shfl_up_sync(0xffffffffu, a.take, d), __shfl_up_sync(0xffffffffu, a.gone, d)};
}

// One thread-block cluster. Every block scans all requests by itself (new tokens, pages taken, pages given back:
// three exclusive sums in request order), so no block waits for another to know where its tokens lie; the blocks
// then share the tokens. The one cluster barrier separates the reads of the old state (lengths, count, table rows
// of finished requests) and the pages pushed on the free stack from the writes of the new state and the pops, which
// is what lets the outputs be the inputs' own buffers. Bound by its chain of dependent loads and barriers, not by
// the 16 bytes written per token: 7.1 us for 256 requests with one token each, 9.2 us for 34,487 tokens of 96 requests
// on a cluster of 8.
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(PagePlanParams p) {
  extern __shared__ int plan_smem[];
  int* s_cu = plan_smem;                           // [B+1] first token of a request
  int* s_old = s_cu + p.B + 1;                     // [B]   tokens kept from before
  int* s_pg = s_old + p.B;                         // [B]   pages taken by the requests before it
  int* s_go = s_pg + p.B;                          // [B+1] pages given back by the requests before it
  __shared__ PlanSums s_warp[PLAN_THREADS / 32];
  __shared__ int s_narrow, s_bad;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P1 = (1 << p.shift) - 1;
  if (tid == 0) { s_narrow = 0; s_bad = 0; }
  __syncthreads();

  const int per = (p.B + PLAN_THREADS - 1) / PLAN_THREADS;
  const int b0 = tid * per, b1 = min(p.B, b0 + per);
  PlanSums mine = {0, 0, 0};
  int narrow = 0, bad = 0;
  auto request = [&](int b, long long& q, long long& old, long long& take, long long& gone) {
    const long long len = max(p.kv_len[b], 0);
    const bool done = p.finished != nullptr && p.finished[b] != 0;
    q = max(p.q_len[b], 0);
    old = done ? 0 : len;
    gone = done ? (len + P1) >> p.shift : 0;
    take = ((old + q + P1) >> p.shift) - ((old + P1) >> p.shift);
  };
  for (int b = b0; b < b1; ++b) {
    long long q, old, take, gone;
    request(b, q, old, take, gone);
    mine.q += q; mine.take += take; mine.gone += gone;
    if ((old + q + P1) >> p.shift > p.W) ++narrow;
    if (gone > p.W) bad = 1;
  }
  PlanSums inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const PlanSums o = plan_shfl_up(inc, d);
    if (lane >= d) { inc.q += o.q; inc.take += o.take; inc.gone += o.gone; }
  }
  if (lane == 31) s_warp[warp] = inc;
  if (narrow) atomicAdd(&s_narrow, narrow);
  if (bad) s_bad = 1;
  __syncthreads();
  if (warp == 0) {
    PlanSums w = s_warp[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const PlanSums o = plan_shfl_up(w, d);
      if (lane >= d) { w.q += o.q; w.take += o.take; w.gone += o.gone; }
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const PlanSums total = s_warp[PLAN_THREADS / 32 - 1];
  const PlanSums before = warp > 0 ? s_warp[warp - 1] : PlanSums{0, 0, 0};
  const long long count = *p.free_count;
  const bool broken = s_bad != 0 || count < 0 || count + total.gone > p.num_pages;
  const long long lack = total.take - count - total.gone, over = total.q - p.capacity;
  const bool ok = !broken && lack <= 0 && over <= 0 && s_narrow == 0;

  {
    PlanSums run = {before.q + inc.q - mine.q, before.take + inc.take - mine.take, before.gone + inc.gone - mine.gone};
    for (int b = b0; b < b1; ++b) {
      long long q, old, take, gone;
      request(b, q, old, take, gone);
      s_cu[b] = ok ? (int)run.q : 0;
      s_old[b] = (int)old;
      s_pg[b] = (int)run.take;
      s_go[b] = ok ? (int)run.gone : 0;
      run.q += q; run.take += take; run.gone += gone;
    }
    if (tid == 0) {
      s_cu[p.B] = ok ? (int)total.q : 0;
      s_go[p.B] = ok ? (int)total.gone : 0;
    }
  }
  __syncthreads();
  // the pages of finished requests go on top of the stack, one warp of the cluster per request
  for (int b = blockIdx.x * (PLAN_THREADS / 32) + warp; b < p.B; b += gridDim.x * (PLAN_THREADS / 32)) {
    const int first = s_go[b], n = s_go[b + 1] - first;
    for (int j = lane; j < n; j += 32) p.free_pages[count + first + j] = p.table[(int64_t)b * p.table_st + j];
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // new state, one block
  if (blockIdx.x == 0) {
    for (int b = tid; b < p.B; b += PLAN_THREADS) {
      p.cu_q[b] = s_cu[b];
      const int now = ok ? s_old[b] + (s_cu[b + 1] - s_cu[b]) : p.kv_len[b];
      p.kv_len_out[b] = now;
    }
    if (tid == 0) {
      p.cu_q[p.B] = s_cu[p.B];
      *p.free_count_out = (int)(ok ? count + total.gone - total.take : count);
      p.status[0] = (int)min(max(lack, 0ll), 0x7fffffffll);
      p.status[1] = (int)min(max(over, 0ll), 0x7fffffffll);
      p.status[2] = s_narrow;
      p.status[3] = broken ? 1 : 0;
    }
  }
  const int live = s_cu[p.B];
  const long long top = count + total.gone - 1;
  for (int n = blockIdx.x * PLAN_THREADS + tid; n < p.capacity; n += gridDim.x * PLAN_THREADS) {
    int64_t slot = -1;
    int pos = -1, b = -1;
    if (n < live) {
      int lo = 0, hi = p.B - 1;                    // last request whose first token is <= n
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_cu[mid] <= n) lo = mid; else hi = mid - 1;
      }
      b = lo;
      pos = s_old[b] + (n - s_cu[b]);
      const int lp = pos >> p.shift, have = (s_old[b] + P1) >> p.shift;
      int page;
      if (lp < have) {
        page = __ldcg(p.table + (int64_t)b * p.table_st + lp);
      } else {
        page = __ldcg(p.free_pages + (top - s_pg[b] - (lp - have)));
        if ((pos & P1) == 0) p.table[(int64_t)b * p.table_st + lp] = page;    // its first row is always new
      }
      if (page >= 0 && page < p.num_pages) slot = ((int64_t)page << p.shift) + (pos & P1);
    }
    p.slot[n] = slot;
    p.position[n] = pos;
    p.request[n] = b;
  }
}

struct PagedAppendParams {
  const uint8_t* key; int64_t k_st, k_sh;          // bytes
  const uint8_t* value; int64_t v_st, v_sh;
  const int64_t* slot; int N, Hkv;
  uint8_t* kpool; int64_t kp_sp, kp_sh, kp_st;     // bytes
  uint8_t* vpool; int64_t vp_sp, vp_sh, vp_st;
  int64_t rows; int shift;                          // rows of the pool: num_pages << shift
};

constexpr int APPEND_THREADS = 256;

// Copies K and V rows to their places: threadIdx.x walks a row in 16-byte pieces, threadIdx.y the (token, head)
// pairs. Bound by HBM: two reads and two writes of a row each, nothing is touched twice: 16083 rows of 8 heads (132 MB) in
// 23.1 us = 5.7 TB/s, 0.87 of the copy bandwidth; 16 rows 1.6 us.
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(PagedAppendParams p) {
  const int64_t pairs = (int64_t)p.N * p.Hkv;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  const int64_t off = (int64_t)threadIdx.x * 16;
  for (int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; r < pairs; r += step) {
    const int n = (int)(r / p.Hkv), h = (int)(r - (int64_t)n * p.Hkv);
    const int64_t slot = p.slot[n];
    if (slot < 0 || slot >= p.rows) {
      if (slot != -1) atomicExch(&g_device_status, (int)KVB_BAD_ARG);
      continue;
    }
    const int64_t page = slot >> p.shift, row = slot & (((int64_t)1 << p.shift) - 1);
    const uint4 k = __ldcs(reinterpret_cast<const uint4*>(p.key + n * p.k_st + h * p.k_sh + off));
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p.value + n * p.v_st + h * p.v_sh + off));
    *reinterpret_cast<uint4*>(p.kpool + page * p.kp_sp + h * p.kp_sh + row * p.kp_st + off) = k;
    *reinterpret_cast<uint4*>(p.vpool + page * p.vp_sp + h * p.vp_sh + row * p.vp_st + off) = v;
  }
}

static inline bool page_tokens_ok(int P) { return P >= 1 && P <= (1 << 24) && (P & (P - 1)) == 0; }
static inline int log2_int(int v) { int s = 0; while ((1 << s) < v) ++s; return s; }

}  // namespace kvb

extern "C" __attribute__((visibility("default"))) int kvb_page_plan(
    const int32_t* kv_len, const int32_t* q_len, const uint8_t* finished, int B, int32_t* page_table,
    int64_t page_table_stride, int W, int32_t* free_pages, int num_pages, const int32_t* free_count, int page_tokens,
    int capacity, int32_t* cu_q, int32_t* kv_len_out, int32_t* free_count_out, int64_t* slot, int32_t* position,
    int32_t* request, int32_t* status, int device, void* stream) {
  using namespace kvb;
  if (!kv_len || !q_len || !page_table || !free_pages || !free_count || !cu_q || !kv_len_out || !free_count_out ||
      !slot || !position || !request || !status)
    return KVB_BAD_ARG;
  if (B < 1 || B > PLAN_MAX_B || W < 1 || num_pages < 1 || capacity < 1 || capacity > (1 << 30) ||
      page_table_stride < W || !page_tokens_ok(page_tokens) || (int64_t)W * page_tokens > 0x40000000)
    return KVB_BAD_SHAPE;
  if (!aligned_to(slot, 8)) return KVB_BAD_ALIGN;
  DeviceGuard guard(device);
  if (!guard.ok) return KVB_BAD_DEVICE;
  const size_t smem = ((size_t)4 * B + 2) * sizeof(int);
  static std::atomic<bool> done[KVB_MAX_DEVICES];
  const int rc = ensure_dynamic_smem(page_plan_kernel, done, device, ((size_t)4 * PLAN_MAX_B + 2) * sizeof(int));
  if (rc != KVB_OK) return rc;
  int ctas = 1;
  while (ctas < PLAN_MAX_CTAS && ctas * PLAN_THREADS < capacity) ctas *= 2;
  PagePlanParams p{kv_len, q_len, finished, B, page_table, page_table_stride, W, free_pages, num_pages, free_count,
                   log2_int(page_tokens), capacity, cu_q, kv_len_out, free_count_out, slot, position, request, status};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(PLAN_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KVB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, page_plan_kernel, p));
  return KVB_OK;
}

extern "C" __attribute__((visibility("default"))) int kvb_paged_append(
    const void* key, int64_t k_st, int64_t k_sh, const void* value, int64_t v_st, int64_t v_sh, const int64_t* slot,
    int N, int Hkv, int D, void* key_pool, int64_t kp_sp, int64_t kp_sh, int64_t kp_st, void* value_pool, int64_t vp_sp,
    int64_t vp_sh, int64_t vp_st, int num_pages, int page_tokens, int device, void* stream) {
  using namespace kvb;
  if (!key || !value || !slot || !key_pool || !value_pool) return KVB_BAD_ARG;
  if (N < 0 || Hkv < 1 || D < 8 || D > 1024 || D % 8 || num_pages < 1 || !page_tokens_ok(page_tokens)) return KVB_BAD_SHAPE;
  const int64_t strides[] = {k_st, k_sh, v_st, v_sh, kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st};
  for (int64_t s : strides)
    if (s % 8 || s < 0) return KVB_BAD_ALIGN;
  if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(key_pool, 16) || !aligned_to(value_pool, 16) ||
      !aligned_to(slot, 8))
    return KVB_BAD_ALIGN;
  DeviceGuard guard(device);
  if (!guard.ok) return KVB_BAD_DEVICE;
  if (N == 0) return KVB_OK;
  const int shift = log2_int(page_tokens);
  PagedAppendParams p{static_cast<const uint8_t*>(key), 2 * k_st, 2 * k_sh, static_cast<const uint8_t*>(value), 2 * v_st,
                      2 * v_sh, slot, N, Hkv, static_cast<uint8_t*>(key_pool), 2 * kp_sp, 2 * kp_sh, 2 * kp_st,
                      static_cast<uint8_t*>(value_pool), 2 * vp_sp, 2 * vp_sh, 2 * vp_st, (int64_t)num_pages << shift, shift};
  const int tx = D / 8, ty = tx >= APPEND_THREADS ? 1 : APPEND_THREADS / tx;
  const int64_t pairs = (int64_t)N * Hkv;
  const int64_t want = (pairs + ty - 1) / ty;
  const int64_t most = (int64_t)sm_count(device) * 32;
  KVB_CHECK_CUDA(launch_kernel(paged_append_kernel, dim3((unsigned)(want < most ? want : most)), dim3(tx, ty), 0,
                               static_cast<cudaStream_t>(stream), p));
  return KVB_OK;
}
