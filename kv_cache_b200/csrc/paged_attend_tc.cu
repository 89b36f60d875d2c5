// Attention over paged K/V for chunks of new tokens, on the 5th-generation tensor cores. Scores, visible ranges, spans
// and pieces: paged_common.cuh.
#include "paged_common.cuh"
#include "tcgen05.cuh"

#include <cuda.h>

#include <type_traits>

namespace kvb {

constexpr int PT_ROWS = 256;                // rows of a unit: two accumulator tiles of 128
constexpr int PT_MAX_GRID = 148;            // one block per SM
constexpr int PT_SNAP = 1, PT_LEAST = 1;    // key tiles, see paged_common.cuh: a short call (2 prompts, 333 tokens) takes 22.8 us,
                                            // 25.7 with 2 and 3, 34.7 with 3 and 5; long ones do not differ
constexpr int PT_KT = 128;                  // keys per tile
constexpr int PT_THREADS = 384;             // warps 0-3, 4-7: softmax of row tile 0, 1; 8, 9: loads; 10: MMA issue
constexpr int PT_HALF = 128 * 128;          // bytes of 128 rows x 64 16-bit elements, 128-byte swizzle
constexpr float PT_LAZY = 8.0f;             // a row's reference moves when a score passes it by 2^8

template <int D>
struct PtCfg {
  static constexpr int NH = D / 64;                      // 64-element halves of a row
  static constexpr int TILEB = NH * PT_HALF;             // one 128-row operand tile
  static constexpr int ST = D == 128 ? 5 : 8;            // K/V ring stages
  static constexpr int QS = D == 128 ? 2 : 4;            // query tiles held; with 4 the next unit's are loaded under this one
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = QS * TILEB;
  static constexpr int OFF_BAR = OFF_KV + ST * TILEB;
  static constexpr int Q_FULL = OFF_BAR, Q_EMPTY = Q_FULL + 8 * QS, FULL = Q_EMPTY + 8 * QS, EMPTY = FULL + 8 * ST;   // barriers
  static constexpr int S_FULL = EMPTY + 8 * ST, P_FULL = S_FULL + 16, DONE = P_FULL + 32, GO = DONE + 8;   // P_FULL[key half][row tile]
  static constexpr int OFF_MISC = GO + 8;                                                             // tmem base, dead
  static constexpr int BYTES = OFF_MISC + 16;           // the third word stays 0: a wait that must not be cut short
  static constexpr int SMEM = BYTES + 1024;              // the base is brought to a swizzle atom
  static constexpr uint32_t TS = 0, TO = 256;            // tensor memory: scores at 128*w, outputs at 256 + D*w
};

__device__ __forceinline__ uint64_t pt_desc(uint32_t addr16, uint32_t lbo) {
  // address in units of 16 bytes (below 256 KiB: no carry out of its field); 128-byte swizzle, 8-row groups 1024 bytes apart
  constexpr uint32_t hi = (1024 >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | (addr16 | (lbo >> 4) << 16);
}
template <typename T>
__host__ __device__ constexpr uint32_t pt_idesc(int n, bool b_mn_major) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t t, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
      "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, "
      "%25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
      "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]),
      "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t t, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {"
      "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Barriers by shared-memory address (one register instead of two).
__device__ __forceinline__ void pt_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pt_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool pt_elect() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one)::"memory");
  return one != 0;
}
// Wait of at most two seconds that also ends once another role of the block has given up (`dead`: a shared word).
__device__ __forceinline__ bool pt_wait(uint32_t bar, uint32_t parity, uint32_t dead) {
  uint32_t ok, began = 0;
  for (uint32_t i = 0;; ++i) {
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(ok) : "r"(dead) : "memory");
    if (ok) return false;
    uint32_t now;
    asm volatile("mov.u32 %0, %globaltimer_lo;" : "=r"(now));
    if (i == 0) began = now;
    else if (now - began > 2000000000u) break;
  }
  asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(dead), "r"(1u) : "memory");
  atomicExch(&g_device_status, (int)KVB_TIMEOUT);
  return false;
}

// The part of a unit that a block has: key tiles [n0, n1), and those that row tile w works on, [na, nb).
struct PtPiece {
  PagedUnit<PT_ROWS, PT_KT> u;
  int n0, n1;
  bool begins, ends;
  __device__ __forceinline__ void set(const PagedParams& p, const PagedPlace& at, const PagedRequest& r, long long left) {
    u.set(p, r, at.tile);
    n0 = u.t0 + at.k;
    n1 = n0 + (int)min((long long)(u.n - at.k), left);
    begins = at.k == 0;
    ends = n1 == u.t0 + u.n;
  }
  __device__ __forceinline__ void rows(const PagedParams& p, const PagedPlace& at, const PagedRequest& r, int w, int& na,
                                       int& nb) const {
    na = nb = n0;
    const int f0 = at.tile * PT_ROWS + w * 128;
    if (f0 >= r.q * p.G) return;
    const int lo = paged_lo(r, p.window, paged_token(p, f0)), hi = paged_hi(r, min(r.q - 1, paged_token(p, f0 + 127)));
    if (hi <= lo) return;
    const int a = max(n0, lo / PT_KT), b = min(n1, (hi + PT_KT - 1) / PT_KT);
    if (a < b) { na = a; nb = b; }
  }
};

// ---- loads: 2 warps ---------------------------------------------------------------------------------------
// The first warp copies by TMA what can be copied as it is: key tiles whose rows all hold tokens of the request, one box
// per page and 64-element half (a page id out of range: a box beyond the pool, which the engine fills with zeros), and
// query tiles when the heads of a KV head divide 128 (a box of 128 / G tokens x G heads is the tile, row by row). The
// rest (the ends of a key range, pages of fewer than 8 tokens, other groups) is copied by both warps, 64 rows each,
// 16 bytes per lane, with zeros for the rows that are not seen.
template <typename T, int D>
struct PtLoader {
  using Cfg = PtCfg<D>;
  static constexpr int CPR = D / 8, RPI = 32 / CPR;
  const PagedParams& p;
  const CUtensorMap* kmap;
  const CUtensorMap* vmap;
  const CUtensorMap* qmap;
  uint32_t base;
  int w, lane;
  int item, qitem;                                       // K/V tiles and query tiles so far
  int rows, goes;                                        // tiles copied by rows and not handed over yet; times the warps met

  __device__ __forceinline__ PtLoader(const PagedParams& p_, const CUtensorMap* k_, const CUtensorMap* v_, const CUtensorMap* q_,
                                      uint32_t base_, int w_, int lane_)
      : p(p_), kmap(k_), vmap(v_), qmap(q_), base(base_), w(w_), lane(lane_), item(0), qitem(0), rows(0), goes(0) {}

  __device__ __forceinline__ bool wait(uint32_t off, uint32_t parity) { return pt_wait(base + off, parity, base + Cfg::OFF_MISC + 4); }
  __device__ __forceinline__ bool wait_empty() { return wait(Cfg::EMPTY + 8 * (item % Cfg::ST), ((item / Cfg::ST) & 1) ^ 1); }
  __device__ __forceinline__ uint32_t stage() const { return base + Cfg::OFF_KV + (item % Cfg::ST) * Cfg::TILEB; }
  __device__ __forceinline__ void signal(uint32_t off) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) pt_arrive(base + off);
  }
  // the arrivals of both warps, and the bytes of one operand tile
  __device__ __forceinline__ void expect(uint32_t bar) {
    if (lane == 0) {
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 1;" ::"r"(bar) : "memory");
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((uint32_t)Cfg::TILEB) : "memory");
    }
    __syncwarp();
  }
  __device__ __forceinline__ bool whole(const PtPiece& pc, int kv, int n) const {
    return p.box > 0 && n * PT_KT >= pc.u.lo && n * PT_KT + PT_KT <= kv && n * PT_KT < pc.u.hi;
  }
  __device__ __forceinline__ void load_boxes(const CUtensorMap* map, int h, int n, int pg) {
    const uint32_t bar = base + Cfg::FULL + 8 * (item % Cfg::ST);
    expect(bar);
    if (lane < PT_KT / p.box) {
      const int row = (n * PT_KT + lane * p.box) & ((1 << p.shift) - 1);
#pragma unroll
      for (int half = 0; half < Cfg::NH; ++half)
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(stage() + half * PT_HALF + lane * p.box * 128), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(half * 64),
            "r"(row), "r"(h), "r"(pg)
            : "memory");
    }
  }
  __device__ __forceinline__ void load_rows(const T* pool, int64_t sp, int64_t st, int n, int pg0, int pg1) {
    const int c = lane % CPR, mask = (1 << p.shift) - 1;
    const uint32_t col = stage() + (c >> 3) * PT_HALF;
#pragma unroll 4
    for (int j = 0; j < 64 / RPI; ++j) {
      const int row = lane / CPR + j * RPI, ra = 64 * w + row;
      const int g = __shfl_sync(0xffffffffu, j < 32 / RPI ? pg0 : pg1, row & 31);
      const bool ok = g >= 0;
      const int64_t at = ok ? (int64_t)g * sp + (int64_t)((n * PT_KT + ra) & mask) * st + c * 8 : 0;
      cp_async_16_or_zero(col + ra * 128 + (((c & 7) ^ (ra & 7)) << 4), pool + at, ok);
    }
    cp_async_commit();
  }
  // requests the K and V rows of key tile n; `pg`: the page of this lane's box when the tile is whole
  __device__ __forceinline__ bool load_tile(const PtPiece& pc, int kv, int n, int h, const int32_t* table, int pg) {
    if (whole(pc, kv, n)) {
      if (w == 0) {
#pragma unroll 1
        for (int i = 0; i < 2; ++i, ++item) {
          if (!wait_empty()) return false;
          load_boxes(i == 0 ? kmap : vmap, h, n, pg);
        }
      } else {
        item += 2;
      }
      return true;
    }
    // Both warps meet here: the second has not waited for the stages of the tiles in between, and a barrier's phases
    // tell apart only neighbouring uses.
    if (lane == 0) pt_arrive(base + Cfg::GO);
    if (!wait(Cfg::GO, goes & 1)) return false;
    ++goes;
    int mine[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = n * PT_KT + 64 * w + 32 * i + lane;
      mine[i] = -1;
      if (t >= pc.u.lo && t < pc.u.hi) {
        mine[i] = table[t >> p.shift];
        if (mine[i] < 0 || mine[i] >= p.num_pages) {
          atomicExch(&g_device_status, (int)KVB_BAD_ARG);
          mine[i] = -1;
        }
      }
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i, ++item, ++rows) {
      if (!wait_empty()) return false;
      if (i == 0) load_rows(reinterpret_cast<const T*>(p.key) + (int64_t)h * p.k_sh, p.k_sp, p.k_st, n, mine[0], mine[1]);
      else load_rows(reinterpret_cast<const T*>(p.value) + (int64_t)h * p.v_sh, p.v_sp, p.v_st, n, mine[0], mine[1]);
    }
    return true;
  }
  // requests the unit's query rows, `tiles` row tiles
  __device__ __forceinline__ bool load_query(const PagedPlace& at, const PagedRequest& r, int tiles) {
    const int total = r.q * p.G;
    for (int tl = 0; tl < tiles; ++tl) {
      const int slot = (qitem + tl) % Cfg::QS, f0 = at.tile * PT_ROWS + tl * 128;
      const uint32_t dst = base + Cfg::OFF_Q + slot * Cfg::TILEB;
      if (p.qbox > 0 && w > 0) continue;
      if (!wait(Cfg::Q_EMPTY + 8 * slot, (((qitem + tl) / Cfg::QS) & 1) ^ 1)) return false;
      if (p.qbox > 0) {
        const uint32_t bar = base + Cfg::Q_FULL + 8 * slot;
        expect(bar);
        if (lane < Cfg::NH)
          asm volatile(
              "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
              ::"r"(dst + lane * PT_HALF), "l"(reinterpret_cast<uint64_t>(qmap)), "r"(bar), "r"(lane * 64), "r"(at.h * p.G),
              "r"(r.first + f0 / p.G)
              : "memory");
        continue;
      }
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int r0 = 64 * w + 32 * half, flat = f0 + r0 + lane;
        int64_t off = -1;
        if (flat < total) {
          const int token = paged_token(p, flat), head = at.h * p.G + (flat - token * p.G);
          off = (int64_t)(r.first + token) * p.q_st + (int64_t)head * p.q_sh;
        }
        const int c = lane % CPR;
        const uint32_t col = dst + (c >> 3) * PT_HALF;
#pragma unroll 4
        for (int j = 0; j < 32 / RPI; ++j) {
          const int row = lane / CPR + j * RPI, ra = r0 + row;
          const int64_t o = __shfl_sync(0xffffffffu, off, row);
          const bool ok = o >= 0;
          cp_async_16_or_zero(col + ra * 128 + (((c & 7) ^ (ra & 7)) << 4), reinterpret_cast<const T*>(p.q) + (ok ? o + c * 8 : 0), ok);
        }
      }
    }
    if (p.qbox == 0) cp_async_commit();
    return true;
  }
  // hands over what was copied by rows: the query tiles, when they were, and the K and V rows of the last tile
  __device__ __forceinline__ void finish(int queries) {
    if (p.qbox > 0) queries = 0;
    if (queries == 0 && rows == 0) return;
    cp_async_wait<0>();
    for (int i = 0; i < queries; ++i) signal(Cfg::Q_FULL + 8 * ((qitem + i) % Cfg::QS));
    if (rows > 0) {
      signal(Cfg::FULL + 8 * ((item - 2) % Cfg::ST));
      signal(Cfg::FULL + 8 * ((item - 1) % Cfg::ST));
      rows = 0;
    }
  }
  __device__ __forceinline__ void run(PagedPlace at, PagedRequest r, long long left) {
    bool ok = true;
    while (ok) {
      PtPiece pc;
      pc.set(p, at, r, left);
      const int32_t* table = p.table + (int64_t)at.b * p.table_st;
      auto box_page = [&](int n) -> int {                // the page of this lane's box of a whole tile
        if (w > 0 || n >= pc.n1 || !whole(pc, r.kv, n) || lane >= PT_KT / p.box) return 0;
        const int pg = table[(n * PT_KT + lane * p.box) >> p.shift];
        if (pg < 0 || pg >= p.num_pages) {
          atomicExch(&g_device_status, (int)KVB_BAD_ARG);
          return p.num_pages;
        }
        return pg;
      };
      int pg = box_page(pc.n0);
      // The unit's query and first keys are requested together. With two query slots (D = 128) the query has to wait
      // for the last scores of the unit before this one; the first keys go ahead of it.
      const int queries = at.tile * PT_ROWS + 128 < r.q * p.G ? 2 : 1;
      const bool early = Cfg::QS == 4 || qitem == 0;
      ok = !early || load_query(at, r, queries);
      for (int n = pc.n0; n < pc.n1 && ok; ++n) {
        const int next = box_page(n + 1);
        ok = load_tile(pc, r.kv, n, at.h, table, pg);
        if (!ok) break;
        if (n == pc.n0) {
          finish(early ? queries : 0);
          if (!early) {
            ok = load_query(at, r, queries);
            if (ok) finish(queries);
          }
          if (ok) qitem += queries;
        } else {
          finish(0);
        }
        pg = next;
      }
      if (!ok) break;
      left -= pc.n1 - pc.n0;
      if (left <= 0 || !paged_next<PT_ROWS>(p, at, r)) break;
    }
    cp_async_wait<0>();
    if (!ok && w == 0) {                                 // nothing of this block may land after it has left
      for (int i = max(0, item - Cfg::ST); i < item; ++i) pt_wait(base + Cfg::FULL + 8 * (i % Cfg::ST), (i / Cfg::ST) & 1, base + Cfg::OFF_MISC + 8);
      for (int i = max(0, qitem - Cfg::QS); i < qitem; ++i) pt_wait(base + Cfg::Q_FULL + 8 * (i % Cfg::QS), (i / Cfg::QS) & 1, base + Cfg::OFF_MISC + 8);
    }
  }
};

// ---- MMA issue: one warp, one elected lane -----------------------------------------------------------------
// Descriptors differ from a constant only in their address word. The whole warp walks the loop with values that are
// the same in every lane (votes and shuffles say so to the compiler) and elects a lane around each group of products:
// a lane chosen by its number made the compiler branch around every single product (3660 instead of 4420 cycles a tile pair).
template <typename T, int D>
__device__ __forceinline__ void pt_issue(const PagedParams& p, uint32_t base_, uint32_t tmem_, PagedPlace at, PagedRequest r, long long left) {
  using Cfg = PtCfg<D>;
  const uint32_t base = __shfl_sync(0xffffffffu, base_, 0), tmem = __shfl_sync(0xffffffffu, tmem_, 0);
  const uint32_t full = base + Cfg::FULL, empty = base + Cfg::EMPTY, s_full = base + Cfg::S_FULL, p_full = base + Cfg::P_FULL;
  const uint32_t dead = base + Cfg::OFF_MISC + 4;
  constexpr uint32_t id_s = pt_idesc<T>(PT_KT, false), id_o = pt_idesc<T>(D, true);
  uint32_t stage = 0, phase = 0;                         // of the next K/V tile
  uint32_t qslot[2] = {0, 0}, qaddr[2] = {0, 0}, qnext = 0, qphase = 0, p_use[2] = {0, 0};
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, pt_wait(bar, parity, dead)); };
  auto commit = [&](uint32_t bar) {
    if (pt_elect()) pt_commit(bar);
    __syncwarp();
  };
  auto step = [&]() { if (++stage == Cfg::ST) { stage = 0; phase ^= 1; } };
  auto scores = [&](int w, uint32_t st) {
    const uint32_t q = qaddr[w], k = (base + Cfg::OFF_KV + st * Cfg::TILEB) >> 4;
    if (pt_elect()) {
#pragma unroll
      for (int h = 0; h < Cfg::NH; ++h)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          pt_mma_ss(tmem + Cfg::TS + 128 * w, pt_desc(q + ((h * PT_HALF + s * 32) >> 4), 16), pt_desc(k + ((h * PT_HALF + s * 32) >> 4), 16),
                    id_s, h + s > 0 ? 1u : 0u);
    }
    __syncwarp();
  };
  while (true) {
    PtPiece pc;
    pc.set(p, at, r, left);
    int na[2], nb[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      pc.rows(p, at, r, w, na[w], nb[w]);
      na[w] = __shfl_sync(0xffffffffu, na[w], 0);
      nb[w] = __shfl_sync(0xffffffffu, nb[w], 0);
    }
    const int n0 = __shfl_sync(0xffffffffu, pc.n0, 0), n1 = __shfl_sync(0xffffffffu, pc.n1, 0);
    const int tiles = __shfl_sync(0xffffffffu, at.tile * PT_ROWS + 128 < r.q * p.G ? 2 : 1, 0);
    // first keys and the query
    bool ok = wait(full + 8 * stage, phase);
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if (w < tiles) {
        ok = ok && wait(base + Cfg::Q_FULL + 8 * qnext, qphase);
        qslot[w] = qnext;
        qaddr[w] = __shfl_sync(0xffffffffu, (base + Cfg::OFF_Q + qnext * Cfg::TILEB) >> 4, 0);
        if (++qnext == Cfg::QS) { qnext = 0; qphase ^= 1; }
      }
    if (!ok) break;
    tc_fence_after();
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if (na[w] == n0 && nb[w] > n0) {
        scores(w, stage);
        commit(s_full + 8 * w);
      }
    if (n0 + 1 == n1) {
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (w < tiles) commit(base + Cfg::Q_EMPTY + 8 * qslot[w]);
    }
    commit(empty + 8 * stage);
    step();
    for (int n = n0; n < n1; ++n) {
      const uint32_t vs = stage, vp = phase;
      step();
      const uint32_t ks = stage;
      const bool more = n + 1 < n1;
      ok = wait(full + 8 * vs, vp) && (!more || wait(full + 8 * ks, phase));
      if (!ok) break;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const bool pv = n >= na[w] && n < nb[w], sc = n + 1 >= na[w] && n + 1 < nb[w];
        if (pv) {
          const uint32_t v = (base + Cfg::OFF_KV + vs * Cfg::TILEB) >> 4;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            ok = ok && wait(p_full + 16 * half + 8 * w, p_use[w] & 1);
            if (ok) {
              tc_fence_after();
              if (pt_elect()) {
#pragma unroll
                for (int j = 4 * half; j < 4 * half + 4; ++j)
                  pt_mma_ts(tmem + Cfg::TO + D * w, tmem + Cfg::TS + 128 * w + 8 * j, pt_desc(v + j * 128, PT_HALF), id_o,
                          (n > na[w] || j > 0) ? 1u : 0u);
              }
              __syncwarp();
            }
          }
          ++p_use[w];
        }
        if (ok && sc) scores(w, ks);
        if (ok && (pv || sc)) commit(s_full + 8 * w);
        if (ok && n + 2 == n1 && w < tiles) commit(base + Cfg::Q_EMPTY + 8 * qslot[w]);      // these were its last scores
      }
      if (!ok) break;
      commit(empty + 8 * vs);
      if (more) {
        commit(empty + 8 * ks);
        step();
      }
    }
    if (!ok) break;
    left -= n1 - n0;
    if (left <= 0 || !paged_next<PT_ROWS>(p, at, r)) break;
  }
  commit(base + Cfg::DONE);
  pt_wait(base + Cfg::DONE, 0, base + Cfg::OFF_MISC + 8);  // no product may run on after tensor memory is given back
}

// ---- softmax of one row tile: 4 warps, one row per thread ------------------------------------------------
template <typename T, int D, bool MOD>
__device__ __forceinline__ void pt_softmax(const PagedParams& p, uint32_t base, uint32_t tmem, int w, int tid, PagedPlace at, PagedRequest r, long long left, long long x,
                                           long long per) {
  using Cfg = PtCfg<D>;
  const uint32_t s_full = base + Cfg::S_FULL + 8 * w, p_full = base + Cfg::P_FULL + 8 * w, dead = base + Cfg::OFF_MISC + 4;
  const int warp = tid >> 5, lane = tid & 31;
  const uint32_t lanes = (uint32_t)(warp * 32) << 16;
  const uint32_t ts = tmem + Cfg::TS + 128 * w + lanes, to = tmem + Cfg::TO + D * w + lanes;
  uint32_t s_use = 0;
  while (true) {
    PtPiece pc;
    pc.set(p, at, r, left);
    int na, nb;
    pc.rows(p, at, r, w, na, nb);
    const int flat = at.tile * PT_ROWS + w * 128 + tid;
    const bool live = flat < r.q * p.G;
    const int token = live ? paged_token(p, flat) : 0, head = at.h * p.G + (live ? flat - token * p.G : 0);
    const int pos = r.kv - r.q + token;
    const int lo = live ? paged_lo(r, p.window, token) : 0, hi = live ? max(lo, paged_hi(r, token)) : 0;
    const float slope = MOD && p.slopes && live ? p.slopes[head] * PA_LOG2E : 0.0f;
    // keys that every row of the tile sees need no mask
    const int f0 = at.tile * PT_ROWS + w * 128;
    const int all_lo = paged_lo(r, p.window, min(r.q - 1, paged_token(p, f0 + 127))), all_hi = paged_hi(r, paged_token(p, f0));
    const bool any = f0 + 32 * warp < r.q * p.G;         // whether the warp has a row at all
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int n = na; n < nb; ++n) {
      if (!pt_wait(s_full, s_use & 1, dead)) { ok = false; break; }
      ++s_use;
      tc_fence_after();
      if (!any) {                                        // what these rows weigh goes nowhere
        if (lane == 0) {
          pt_arrive(p_full);
          pt_arrive(p_full + 16);
        }
        continue;
      }
      // Pass 1: the largest score. Scores that are changed (capped, biased, masked) go back to their place. Reading the
      // tile twice costs less than holding its 128 scores: registers would spill.
      const int t0 = n * PT_KT;
      const bool edge = t0 < all_lo || t0 + PT_KT > all_hi;
      uint32_t v[2][32];
      float mx[2] = {-INFINITY, -INFINITY};
      auto largest = [&](const uint32_t* x) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          asm("max.f32 %0, %0, %1, %2;" : "+f"(mx[0]) : "f"(__uint_as_float(x[i])), "f"(__uint_as_float(x[i + 1])));
          asm("max.f32 %0, %0, %1, %2;" : "+f"(mx[1]) : "f"(__uint_as_float(x[i + 2])), "f"(__uint_as_float(x[i + 3])));
        }
      };
      if (MOD || edge) {
        // a loop, not straight code: a tile would otherwise stream tens of kilobytes of instructions
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          TcLd<32>::ld(ts + 32 * c, v[0]);
          TcLd<32>::wait(v[0]);
          if constexpr (MOD) {
            paged_scale<32>(p, reinterpret_cast<float*>(v[0]));
            if (p.slopes) paged_bias<32>(reinterpret_cast<float*>(v[0]), slope, t0 + 32 * c - pos);
          }
          if (edge) {
            const uint32_t seen = paged_seen(t0 + 32 * c, lo, hi);
            if (__any_sync(0xffffffffu, seen != 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(seen >> i & 1u)) v[0][i] = 0xff800000u;
            }
          }
          tc_st32(ts + 32 * c, v[0]);
          largest(v[0]);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < 4; c += 2) {
          TcLd<32>::ld(ts + 32 * c, v[0]);
          TcLd<32>::ld(ts + 32 * c + 32, v[1]);
          TcLd<32>::wait(v[0]);
          TcLd<32>::wait(v[1]);
          largest(v[0]);
          largest(v[1]);
        }
      }
      if (MOD || edge) tc_wait_st();
      TcLd<32>::ld(ts, v[0]);
      const float scale = MOD ? 1.0f : p.scale_log2;
      const float top = fmaxf(mx[0], mx[1]) * scale;
      const bool move = top > m + PT_LAZY;
      if (__any_sync(0xffffffffu, move)) {
        const float mn = move ? top : m, a = move ? ex2(m - mn) : 1.0f;
        m = mn;
        l *= a;
        if (n > na) {                                    // the product before this one is complete: it was issued before these scores
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            TcLd<32>::ld(to + 32 * c, o);
            TcLd<32>::wait(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
            tc_st32(to + 32 * c, o);
          }
        }
      }
      const float ms = m == -INFINITY ? 0.0f : m;
      // Pass 2: weights, two at a time.
      const uint64_t scale2 = pack2(scale, scale), ms2 = pack2(-ms, -ms);
      constexpr float W = Half2Of<T>::WEIGHT;
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
        TcLd<32>::wait(v[c & 1]);
        if (c < 3) TcLd<32>::ld(ts + 32 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float a, b;
          unpack2(fma2(pack2(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])), scale2, ms2), a, b);
          a = ex2(a);
          b = ex2(b);
          sum[i & 1] = add2(sum[i & 1], pack2(a, b));
          if constexpr (W != 1.0f) unpack2(mul2(pack2(a, b), pack2(W, W)), a, b);
          pk[i] = Half2Of<T>::pack(a, b);
        }
        tc_st16(ts + 16 * c, pk);
        if (c & 1) {                                     // half of the keys: the second product may begin
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) pt_arrive(p_full + 16 * (c >> 1));
        }
      }
      float s0, s1;
      unpack2(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
    }
    if (!ok) return;
    // ---- the unit, or this block's piece of it
    const bool some = nb > na;
    if (some) {
      if (!pt_wait(s_full, s_use & 1, dead)) return;
      ++s_use;
      tc_fence_after();
    }
    const bool whole = pc.begins && pc.ends;
    const int slot = 2 * blockIdx.x + (pc.begins ? 1 : 0);
    constexpr float W = Half2Of<T>::WEIGHT;
    const float inv = (l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l)) * (1.0f / W);
    const int64_t row = (int64_t)(r.first + token) * p.Hq + head;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      if (some) {
        TcLd<32>::ld(to + 32 * c, o);
        TcLd<32>::wait(o);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0u;
      }
      if (!live) continue;
      if (whole) {
        uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + row * D + 32 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = Half2Of<T>::pack(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
          out[i] = make_uint4(x[0], x[1], x[2], x[3]);
        }
      } else {
        uint4* dst = reinterpret_cast<uint4*>(p.ws_o + ((int64_t)slot * PT_ROWS + w * 128 + tid) * D + 32 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (W != 1.0f)
#pragma unroll
            for (int e = 4 * i; e < 4 * i + 4; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * (1.0f / W));
          dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
    }
    if (live) {
      if (!whole) p.ws_ml[(int64_t)slot * PT_ROWS + w * 128 + tid] = make_float2(m, l);
      else if (p.lse) p.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * PA_LN2;
    }
    if (pc.begins && !pc.ends && w == 0 && tid == 0) {
      p.ws_desc[2 * blockIdx.x] = make_int4(paged_pieces(per, x, pc.u.n, PT_SNAP, blockIdx.x), at.h, at.tile, 0);
      p.ws_desc[2 * blockIdx.x + 1] = make_int4(r.first, r.q, 0, 0);
    }
    x += pc.n1 - pc.n0;
    tc_fence_before();                                   // the next unit's product overwrites the output once its weights are signalled
    left -= pc.n1 - pc.n0;
    if (left <= 0 || !paged_next<PT_ROWS>(p, at, r)) return;
  }
}

// Each role walks the span with its own copy: what all three derive from it would otherwise be computed ahead of their
// branches and held, or spilled, through all of them.
__device__ __forceinline__ void pt_own(PagedPlace& at, PagedRequest& r, long long& left) {
  asm volatile("" : "+r"(at.b), "+r"(at.h), "+r"(at.tile), "+r"(at.k), "+r"(r.first), "+r"(r.q), "+r"(r.kv), "+r"(r.pre), "+l"(left));
}

// A block walks its span unit by unit: two warps bring K and V tiles (and each unit's query rows) into shared memory in the
// 128-byte-swizzled layout, one warp issues S_w = Q_w K^T and O_w += P_w V for two row tiles w of 128 rows, and four
// warps per row tile, one row per thread, turn scores into weights: S_w is read from tensor memory, P_w goes back over
// it as 16-bit operand of the second product, and O_w stays in tensor memory until the unit ends. While the softmax of
// one row tile runs, the tensor core works on the other. The reference of a row moves only when a score passes it by
// 2^8, so O_w is rescaled rarely, and then by the softmax warps, which know from the order of issue that the previous
// product is complete. Weights are rounded to the input type for the second product, as the values they weigh are; their
// sum is taken before that. Rows of K and V that no token of the request sees are zero-filled, not read.
//
// 384 threads so that a block's 65536 registers give 208 to a softmax thread and 88 to the others: with
// 512 threads spills in the issuing warp cost a quarter of the time. Measured, bf16: the last 2048 of 32768 tokens, 32/8 heads
// (1.07 TFLOP) 0.94-0.98 ms = 1090-1138 TFLOP/s, 0.66-0.69 of the cuBLAS burst rate (1.07 ms under the power cap): 3650
// cycles per pair of row tiles and key tile, of which the products fill 2048 and the 32768 exponentials, 16 a cycle, 2048.
template <typename T, int D, bool MOD>
__global__ void __launch_bounds__(PT_THREADS, 1)
    paged_chunk_kernel(const __grid_constant__ PagedParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ CUtensorMap qmap) {
  using Cfg = PtCfg<D>;
  extern __shared__ uint8_t pt_raw[];
  const uint32_t raw = smem_u32(pt_raw);
  uint8_t* smem = pt_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t base = smem_u32(smem);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_MISC);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same in all lanes, and known to be
  pdl_launch_dependents();

  const PagedSpan span = paged_span<PT_ROWS, PT_KT, PT_THREADS>(p, reinterpret_cast<int*>(smem + Cfg::OFF_KV), PT_SNAP, PT_LEAST);
  if (tid == 0) p.ws_desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
  if (span.left <= 0) return;
  PagedPlace at = span.at;
  long long left = span.left;
  if (warp == 0) {
    tc_alloc(s_tmem, 512);
    tc_relinquish();
  }
  if (tid == 32) {
    s_tmem[1] = s_tmem[2] = 0;
    auto bar = [&](int off) { return reinterpret_cast<uint64_t*>(smem + off); };
    for (int i = 0; i < Cfg::QS; ++i) {
      mbar_init(bar(Cfg::Q_FULL + 8 * i), 2);
      mbar_init(bar(Cfg::Q_EMPTY + 8 * i), 1);
    }
    for (int i = 0; i < Cfg::ST; ++i) {
      mbar_init(bar(Cfg::FULL + 8 * i), 2);
      mbar_init(bar(Cfg::EMPTY + 8 * i), 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(bar(Cfg::S_FULL + 8 * w), 1);
      mbar_init(bar(Cfg::P_FULL + 8 * w), 4);
      mbar_init(bar(Cfg::P_FULL + 16 + 8 * w), 4);
    }
    mbar_init(bar(Cfg::DONE), 1);
    mbar_init(bar(Cfg::GO), 2);
    fence_mbar_init();
  }
  PagedRequest r = paged_request(p, at.b);
  fence_proxy_async_smem();                              // the scheduler's scratch is written by the TMA engine next
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  // registers: 168 x 384 at launch = 208 x 256 + 88 x 128
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    pt_own(at, r, left);
    pt_softmax<T, D, MOD>(p, base, tmem, warp >> 2, tid & 127, at, r, left, span.x, span.per);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    pt_own(at, r, left);
    if (warp < 10) {
      PtLoader<T, D> loader(p, &kmap, &vmap, &qmap, base, warp - 8, lane);
      loader.run(at, r, left);
    } else if (warp == 10) {
      pt_issue<T, D>(p, base, tmem, at, r, left);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tc_dealloc(tmem, 512);
}

}  // namespace kvb
