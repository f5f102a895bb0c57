// MXFP4 products on tcgen05 block-scaled MMA (sm_100a).
//
// For every group g, row r of its segment and feature m:
//   Y[r, m] = sum_k  W_g[m, k] X[r, k]
// W_g MXFP4; X either bf16 held as two e4m3 terms with shared scales (see
// mxfp4.cuh; kind::mxf8f6f4, W * hi + W * lo) or MXFP4 itself (kind::mxf4).
// The tensor core multiplies both sides' scales in, so the accumulators stay
// in TMEM over the whole of K and are read once per work unit.
//
// Weights are the 128-row operand A, rows of X the N operand, so that few
// rows waste little. A work unit is two A tiles (256 features, or 128 gate and
// the same 128 up features for the SwiGLU form) times one token tile: the
// token tile is read from L2 once for both, and a thread of the epilogue
// holds gate and up of the same feature and token.
//
// 4-bit weights next to 8-bit activations: TMA widens 16 codes (8 bytes) to
// 16 bytes of shared memory (8 bytes of padding), the layout kind::mxf8f6f4
// reads, so a 128-number K block of one row is 128 bytes on both sides.
//
// Warp roles (one CTA per SM, persistent):
//   warp 0     TMA producer (one thread)
//   warps 1, 2 MMA issuers (one thread each; warp 1 also allocates TMEM), one
//              for each A tile: per stage the thread copies the scale atoms to
//              its TMEM columns (tcgen05.cp) and issues the MMAs behind them
//   warp 3     unit planner, a shared-memory ring of decoded units
//   warps 4..  epilogue, 16 warps: lane quadrant w % 4, 8-column chunks. With few
//              rows (RAW) some of them prepare the rows instead, each for one
//              stage of the ring: split bf16 rows into the stage's operand and
//              atom, or gather MXFP4 rows' scales into the atom. What a kernel
//              in front costs, a launch and 1-2 us, is then gone.
// Two issuing threads because one that waits on a barrier between its batches
// leaves the tensor pipe idle: one thread for both tiles ran 512 rows over 256
// experts 5% slower, a T=4096 product 1%. Sharing A between the hi and the lo MMA
// (collector::a) needs one thread and gave back half a percent: not kept.
// TMEM: two halves of accumulator columns, then one set of scale columns per
// stage (a stage's scales are overwritten only after its MMAs released it). A
// unit that fits a half alternates between them, so its epilogue overlaps the
// next unit's MMAs; a larger one takes both.
//
// What bounds it. Few rows: the weights' bytes from HBM (512 rows over 256
// experts of 7168 x 2048: 255 to 259 us, 6.7 TB/s; gate and up of a 64-token FFN
// 570 to 585 us, 6.0 TB/s). Many: the tensor pipe under the power limit. T=4096 x
// 7168 x 18432 takes 680 to 700 us by itself (1545 to 1590 TFLOP/s in useful
// operations, the pipe 89% busy at 1.51 GHz; in long runs the clock falls to 1.17),
// and 4-bit rows x 18432 x 7168 211 us (5.1 PFLOP/s, 66% at 1.65 GHz). A stage's copies take ~2000 cycles from issue to use; three
// stages of 76 KB hide them at 1280 MMA cycles a stage.
#include <atomic>

#include "common.cuh"
#include "mxfp4.cuh"

namespace dsmoe {
namespace mx {
namespace {

constexpr int BM = 128;
constexpr int RING = 4;
constexpr int PLAN_WARP = 3;
constexpr int EPI_WARP0 = 4;
constexpr int CHUNK = 8;
constexpr int THREADS = (EPI_WARP0 + kWorkWarps) * 32;

struct Unit {
  int32_t ncols;   // valid rows of the token tile; 0: no more units
  int32_t row0;    // first row
  int32_t tile;    // token tile index (scale atoms)
  int32_t group;
  int32_t m0, m1;  // first feature of each A tile; m1 < 0: one A tile only
  int32_t n;       // MMA N of one term
  int32_t both;    // hi and lo side by side (N = 2 n)
  int32_t kb0, kb1;
  int32_t part;    // K part
};

template <bool FP4_, int BN_, int STAGES_, bool RAW_ = false>
struct Cfg {
  static constexpr bool FP4 = FP4_;
  static constexpr bool RAW = RAW_;  // the kernel prepares the rows
  static constexpr int EPI = !RAW ? kWorkWarps : FP4 ? 12 : 4;  // epilogue warps
  // Warps that prepare rows, each for one stage (16 bf16 rows of it): a warp that
  // skipped a fill of a stage could take that fill's phase of `empty` for its own.
  static constexpr int PREP_STAGE = !RAW ? 0 : FP4 ? 1 : BN_ / 16;
  static constexpr int PREP = PREP_STAGE * STAGES_;
  static constexpr int NUM_CG = EPI / 4;
  static constexpr int BN = BN_;
  static constexpr int STAGES = STAGES_;
  static constexpr int KB_STAGE = FP4 ? 2 : 1;  // 128-number K blocks per stage (128 bytes of a row)
  static constexpr int TERMS = FP4 ? 1 : 2;
  static constexpr int ATOMS = tile_atoms(BN);
  static constexpr int A_BYTES = BM * 128;
  // What an A tile's copy counts on its mbarrier: the packed bytes it reads,
  // without the padding it writes between them.
  static constexpr int A_TX = FP4 ? A_BYTES : A_BYTES / 2;
  static constexpr int B_OFF = 2 * A_BYTES;
  static constexpr int B_BYTES = TERMS * BN * 128;
  static constexpr int SFA_BYTES = KB_STAGE * 1024;  // both A tiles'
  static constexpr int SFB_BYTES = KB_STAGE * ATOMS * 512;
  // Operand tiles start on 1024 bytes (128-byte swizzle), so the scale atoms
  // of all stages live behind the operands of all stages.
  static constexpr int OP_BYTES = B_OFF + B_BYTES;
  static constexpr int SF_BYTES = SFA_BYTES + SFB_BYTES;
  static constexpr int SF0 = STAGES * OP_BYTES;
  // TMEM columns
  static constexpr int SF_COLS = KB_STAGE * (1 + ATOMS) * 4;  // of one issuer and stage
  static constexpr int SF_TOTAL = STAGES * 2 * SF_COLS;
  static constexpr int HALF = (512 - SF_TOTAL) / 2 / 16 * 16;
  static constexpr int SF_BASE = 2 * HALF;
  static constexpr int CHUNKS = (BN + NUM_CG * CHUNK - 1) / (NUM_CG * CHUNK);  // of an epilogue warp
  static constexpr int BAR_OFF = STAGES * (OP_BYTES + SF_BYTES);
  // full[S], empty[S], tfull[2], tempty[2], done, ufull[RING], uempty[RING]
  static constexpr int NUM_BARS = 2 * STAGES + 5 + 2 * RING;
  static constexpr int MISC_OFF = BAR_OFF + 8 * NUM_BARS;
  static constexpr int PLAN_OFF = (MISC_OFF + 16 + 15) / 16 * 16;
  static constexpr int TAB_OFF = PLAN_OFF + RING * static_cast<int>(sizeof(Unit));
  static constexpr bool OWN = !FP4 && !RAW && BN <= 64;  // builds the group tables of a few rows itself
  // Group tables: kind::mxf4 and RAW have none.
  static constexpr int SMEM = TAB_OFF + (FP4 || RAW ? 0 : OWN ? 4 * (3 * kMaxGroups + 1) : 4 * (kMaxGroups + 1)) + 1024;
  static_assert(SMEM <= 232448, "shared memory");
  static_assert(EPI + PREP <= kWorkWarps, "warps");
  static_assert(STAGES * OP_BYTES >= BN * 2 * BM * 4, "a K part's sums");
  static_assert(OP_BYTES % 1024 == 0, "operand alignment");
  static_assert(HALF >= BN && (FP4 || 4 * (BN < 96 ? BN : 96) <= 2 * HALF), "accumulator columns");
};

__device__ __forceinline__ uint64_t policy_evict_normal() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// Shared memory written by this thread is read by the tensor core next.
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 512-byte scale atom (32 rows of 16 bytes, unswizzled) -> 4 TMEM columns,
// repeated in all four lane quadrants.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t saddr) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 32;  // 8 rows of 16 bytes to the next 8
  d |= static_cast<uint64_t>(1) << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}

template <bool FP4>
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                           uint32_t sfb, uint32_t acc) {
  if constexpr (FP4)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Two floats at this CTA's shared-memory address `p`, read in CTA `rank` of
// the cluster.
__device__ __forceinline__ float2 load_peer(const float* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// Instruction descriptor of the block-scaled kinds: D fp32, both operands
// K-major, e8m0 scales; A e2m1, B e4m3 (mxf8f6f4) or e2m1 (mxf4). sf_id is
// the byte of the 32-bit scale words an MMA's K starts at.
template <bool FP4>
__device__ __forceinline__ uint32_t idesc_scaled(int n) {
  const uint32_t at = FP4 ? 1u : 5u, bt = FP4 ? 1u : 0u;
  return (at << 7) | (bt << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(BM >> 7) << 27);
}
__device__ __forceinline__ constexpr uint32_t sf_id(int sf) {
  return (static_cast<uint32_t>(sf) << 4) | (static_cast<uint32_t>(sf) << 29);
}
struct True { static constexpr bool value = true; };
struct False { static constexpr bool value = false; };

// One thread of a converged warp. The compiler knows that a single thread is
// active behind it, so that descriptors go to uniform registers once.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// The planner's group tables in shared memory: tile_start, and where the kernel
// builds its own also counts and row_start. Unused without groups.
template <class C>
struct Tables {
  int* tiles;  // [kMaxGroups + 1]
  __device__ __forceinline__ int* counts() const { return tiles + kMaxGroups + 1; }
  __device__ __forceinline__ int* starts() const { return counts() + kMaxGroups; }
};

// One warp, from a routing or from offsets: what route_split_kernel and
// segments_split_kernel compute, lane l for groups 16 l and up.
template <class C>
__device__ __forceinline__ void build_tables(const Tables<C>& t, const GemmArgs& p, int lane) {
  constexpr int GL = kMaxGroups / 32;
  int *cnt = t.counts(), *start = t.starts();
  const TableSource& o = p.own;
  if (o.idx) {
    for (int g = lane; g < kMaxGroups; g += 32) cnt[g] = 0;
    __syncwarp();
    for (int i = lane; i < o.pairs; i += 32) {
      const int64_t e = __ldg(o.idx + i);
      if (e >= 0 && e < o.n_routed) atomicAdd(&cnt[e + o.shared], 1);
    }
    __syncwarp();
    if (o.shared && lane == 0) cnt[0] = o.tokens;
    __syncwarp();
  } else {
    const int R = p.g.rows, first = min(max(__ldg(o.offsets), 0), R);
    int end[GL], top = first;
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      const int g = GL * lane + j;
      if (g < p.g.n) top = max(top, min(max(__ldg(o.offsets + g + 1), 0), R));
      end[j] = top;
    }
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, top, s);
      if (lane >= s) top = max(top, a);
    }
    int before = __shfl_up_sync(0xffffffffu, top, 1);
    if (lane == 0) before = first;
#pragma unroll
    for (int j = 0; j < GL; ++j) {
      const int a = j ? max(before, end[j - 1]) : before;
      start[GL * lane + j] = a;
      cnt[GL * lane + j] = max(before, end[j]) - a;
    }
  }
  int rows = 0, tiles = 0;
  for (int j = 0; j < GL; ++j) {
    const int c = cnt[GL * lane + j];
    rows += c;
    tiles += (c + C::BN - 1) / C::BN;
  }
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, rows, s), b = __shfl_up_sync(0xffffffffu, tiles, s);
    if (lane >= s) rows += a, tiles += b;
  }
  if (lane == 31) t.tiles[kMaxGroups] = tiles;
  for (int j = GL - 1; j >= 0; --j) {
    const int c = cnt[GL * lane + j];
    rows -= c;
    tiles -= (c + C::BN - 1) / C::BN;
    if (o.idx) start[GL * lane + j] = rows;
    t.tiles[GL * lane + j] = tiles;
  }
  __syncwarp();
}

template <class C, bool SWIGLU>
__device__ __forceinline__ Unit decode(int u, const GemmArgs& p, const Tables<C>& t, bool own) {
  Unit e;
  const int per = SWIGLU ? (p.M + BM - 1) / BM : (p.M + 2 * BM - 1) / (2 * BM);
  const int id = p.ksplit > 1 ? u / p.ksplit : u;
  e.part = u - id * p.ksplit;
  int g = 0, rows = p.g.rows, row_start = 0, tile0 = 0, ntiles;
  if (p.g.counts) {
    int lo = 0, hi = p.g.n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (t.tiles[mid] * per <= id) lo = mid; else hi = mid;
    }
    g = lo;
    rows = own ? t.counts()[g] : load_dep(p.g.counts + g);
    row_start = own ? t.starts()[g] : load_dep(p.g.row_start + g);
    tile0 = t.tiles[g];
  }
  ntiles = (rows + C::BN - 1) / C::BN;
  const int local = id - tile0 * per;
  const int mt = local / ntiles, nt = local - mt * ntiles;
  e.group = g;
  e.ncols = min(C::BN, rows - nt * C::BN);
  e.row0 = row_start + nt * C::BN;
  e.tile = tile0 + nt;
  e.m0 = mt * (SWIGLU ? BM : 2 * BM);
  e.m1 = SWIGLU ? e.m0 : (e.m0 + BM < p.M ? e.m0 + BM : -1);
  const int n = C::FP4 ? 0 : side_by_side(C::BN, e.ncols);
  e.both = n > 0;
  e.n = n ? n : (e.ncols + 15) & ~15;
  const int KB = p.K / 128;
  e.kb0 = 0;
  e.kb1 = KB;
  if (p.ksplit > 1) {
    // whole stages per part
    const int st = (KB + C::KB_STAGE - 1) / C::KB_STAGE;
    e.kb0 = static_cast<int>(static_cast<long long>(st) * e.part / p.ksplit) * C::KB_STAGE;
    e.kb1 = min(KB, static_cast<int>(static_cast<long long>(st) * (e.part + 1) / p.ksplit) * C::KB_STAGE);
  }
  return e;
}

// Four tokens' bf16 values of 32 features, packed by token pairs (p01: tokens 0
// and 1 of this lane's feature), transposed over groups of 4 lanes: lane l
// gets features (l & ~3) .. + 3 of token l & 3.
__device__ __forceinline__ uint2 transpose4(uint32_t p01, uint32_t p23, int lane) {
  const uint32_t sel = lane & 1 ? 0x3276 : 0x5410;
  const uint32_t a = __byte_perm(p01, __shfl_xor_sync(0xffffffffu, p01, 1), sel);
  const uint32_t b = __byte_perm(p23, __shfl_xor_sync(0xffffffffu, p23, 1), sel);
  const uint32_t o = __shfl_xor_sync(0xffffffffu, lane & 2 ? a : b, 2);
  return lane & 2 ? make_uint2(o, b) : make_uint2(a, o);
}
// The same for four tokens' bytes.
__device__ __forceinline__ uint32_t transpose4(uint32_t v, int lane) {
  v = __byte_perm(v, __shfl_xor_sync(0xffffffffu, v, 1), lane & 1 ? 0x3715 : 0x6240);
  return __byte_perm(v, __shfl_xor_sync(0xffffffffu, v, 2), lane & 2 ? 0x3276 : 0x5410);
}

template <class C, bool SWIGLU>
__global__ void __launch_bounds__(THREADS, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap tm_w0, const __grid_constant__ CUtensorMap tm_w1,
               const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_x32,
               const __grid_constant__ CUtensorMap tm_x8, const GemmArgs p) {
  constexpr bool FP4 = C::FP4;
  constexpr int BN = C::BN, STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* done_bar = tempty + 2;
  uint64_t* ufull = done_bar + 1;
  uint64_t* uempty = ufull + RING;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::MISC_OFF);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::MISC_OFF + 4);
  Unit* plan = reinterpret_cast<Unit*>(smem + C::PLAN_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1 + C::PREP_STAGE);  // producer, the warps that prepare the stage's rows
      mbar_init(&empty[s], 2);  // both issuers
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 2);
      mbar_init(&tempty[b], C::EPI);
    }
    mbar_init(done_bar, 2);
    for (int r = 0; r < RING; ++r) {
      mbar_init(&ufull[r], 1);
      mbar_init(&uempty[r], 3 + C::EPI + C::PREP);  // producer, issuers, epilogue and preparing warps
    }
    *s_abort = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_w0);
    prefetch_tmap(&tm_w1);
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_x32);
    prefetch_tmap(&tm_x8);
  }
  if (warp == 1) tmem_alloc(s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  launch_dependents();
  // With group tables of an earlier kernel of the chain every role waits for
  // it. Without, only the copies of the rows do: the producer waits, after it
  // has started on the weights.
  const bool own = C::OWN && (p.own.idx || p.own.offsets);
  const bool early = !p.g.counts || own;
  if (!early) dependency_wait();
  const uint32_t tmem = *s_tmem;
  const int KB = p.K / 128;

  if (warp == PLAN_WARP) {
    // ------------------------------------------------------------- planner
    // The search for a unit's group walks a shared-memory copy of the table:
    // nine dependent global loads would be ~3 us before the first copy.
    const Tables<C> tab{reinterpret_cast<int*>(smem + C::TAB_OFF)};
    int tiles = (p.g.rows + BN - 1) / BN;
    if (p.g.counts) {
      if (own) {
        if constexpr (C::OWN) build_tables<C>(tab, p, lane);
      } else {
        for (int t = lane; t <= p.g.n; t += 32) tab.tiles[t] = load_dep(p.g.tile_start + t);
        __syncwarp();
      }
      tiles = tab.tiles[p.g.n];
    }
    const int total = p.ksplit > 1 ? p.unit0 + static_cast<int>(gridDim.x)
                                   : tiles * (SWIGLU ? (p.M + BM - 1) / BM : (p.M + 2 * BM - 1) / (2 * BM));
    if (lane == 0) {
      int u = p.unit0 + static_cast<int>(blockIdx.x);
      for (int i = 0;; ++i) {
        Unit e;
        e.ncols = 0;  // the end
        if (u < total) e = decode<C, SWIGLU>(u, p, tab, own);
        const int ri = i % RING;
        if (!mbar_wait(&uempty[ri], ((i / RING) & 1) ^ 1, p.status, kDevTimeoutProducer, s_abort)) break;
        plan[ri] = e;
        mbar_arrive(&ufull[ri]);
        // Also in a CTA without a unit, so that this kernel does not end before
        // its predecessor; and before p.next, which an earlier kernel clears.
        if (i == 0 && own) dependency_wait();
        if (u >= total) break;
        // Units of ragged groups cost between 64 and 160 columns: handed out
        // as CTAs become free. (In fixed turns the slowest of 148 CTAs got
        // ~20% more than the mean.)
        u = p.next ? static_cast<int>(gridDim.x) + atomicAdd(p.next, 1) : u + static_cast<int>(gridDim.x);
      }
    }
  } else if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      // Rows are read by every feature tile: kept. Weights: where experts have
      // few rows a weight tile is read once or twice and makes room first;
      // with large token tiles the lines its 64-byte reads promote must outlive
      // the other CTAs' rows (evict-first: 1.5-4% slower).
      const uint64_t pol_w = BN > 64 ? policy_evict_normal() : policy_evict_first(), pol_x = policy_evict_last();
      int stage = 0, issued = 0, i = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (; ok; ++i) {
        const int ri = i % RING;
        if (!mbar_wait(&ufull[ri], (i / RING) & 1, p.status, kDevTimeoutProducer, s_abort)) break;
        const Unit e = plan[ri];
        if (e.ncols == 0) break;
        mbar_arrive(&uempty[ri]);
        const int wrow = e.group * p.M;
        const bool two = e.m1 >= 0;
        const int pairs = SWIGLU ? p.M / BM : (p.M + 2 * BM - 1) / (2 * BM);
        const uint8_t* fa = p.sfa + (static_cast<size_t>(e.group) * pairs + e.m0 / (SWIGLU ? BM : 2 * BM)) * KB * 1024;
        const uint8_t* fb = p.sfb + static_cast<size_t>(e.tile) * KB * (C::ATOMS * 512);
        const uint32_t xbytes = C::RAW && !FP4 ? 0 : e.both ? 2 * e.n * 128 : C::B_BYTES;
        auto load_w = [&](int kb, int stage) {
          uint8_t* st = smem + stage * C::OP_BYTES;
          uint8_t* sf = smem + C::SF0 + stage * C::SF_BYTES;
          const int nkb = min(C::KB_STAGE, e.kb1 - kb);  // an odd last K block: only its scales exist
          const int kx = FP4 ? kb * 64 : kb * 128;  // coordinate: bytes of packed codes, or numbers
          mbar_arrive_expect_tx(&full[stage], (two ? 2 : 1) * C::A_TX + nkb * 1024 + xbytes + (C::RAW ? 0 : nkb * C::ATOMS * 512));
          tma_load_2d(st, &tm_w0, &full[stage], kx, wrow + e.m0, pol_w);
          if (two) tma_load_2d(st + C::A_BYTES, &tm_w1, &full[stage], kx, wrow + e.m1, pol_w);
          bulk_load(sf, fa + static_cast<size_t>(kb) * 1024, nkb * 1024, &full[stage]);
        };
        auto load_x = [&](int kb, int stage) {
          if (C::RAW && !FP4) return;
          uint8_t* st = smem + stage * C::OP_BYTES + C::B_OFF;
          const int nkb = min(C::KB_STAGE, e.kb1 - kb);
          const int kx = FP4 ? kb * 64 : kb * 128;
          if (!FP4 && e.both) {
            // 32-row boxes and 8-row boxes for the rest (64 rows instead of 16
            // per stage took a tenth of a one-token FFN).
            for (int s = 0, step; s < e.n; s += step) {
              step = e.n - s >= 32 ? 32 : 8;
              const CUtensorMap* tm = step == 32 ? &tm_x32 : &tm_x8;
              tma_load_2d(st + s * 128, tm, &full[stage], kx, e.row0 + s, pol_x);
              tma_load_2d(st + (e.n + s) * 128, tm, &full[stage], kx, p.P + e.row0 + s, pol_x);
            }
          } else {
            tma_load_2d(st, &tm_x, &full[stage], kx, e.row0, pol_x);
            if (!FP4) tma_load_2d(st + BN * 128, &tm_x, &full[stage], kx, p.P + e.row0, pol_x);
          }
          if (C::RAW) return;
          bulk_load(smem + C::SF0 + stage * C::SF_BYTES + C::SFA_BYTES,
                    fb + static_cast<size_t>(kb) * (C::ATOMS * 512), nkb * C::ATOMS * 512, &full[stage]);
        };
        int kb = e.kb0;
        if (i == 0 && early) {
          // The first stages' weights are on their way while the kernel before
          // this one still prepares the rows.
          const int n = min(STAGES, (e.kb1 - kb + C::KB_STAGE - 1) / C::KB_STAGE);
          for (int s = 0; s < n; ++s) load_w(kb + s * C::KB_STAGE, s);
          dependency_wait();
          for (int s = 0; s < n; ++s) load_x(kb + s * C::KB_STAGE, s);
          issued = n;
          kb += n * C::KB_STAGE;
          stage = n % STAGES;
          phase = n == STAGES;
        }
        for (; kb < e.kb1; kb += C::KB_STAGE) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.status, kDevTimeoutProducer, s_abort)) { ok = false; break; }
          load_w(kb, stage);
          load_x(kb, stage);
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // The last copies must have landed before the CTA may exit.
      const int n_drain = issued < STAGES ? issued : STAGES;
      for (int d = 0; d < n_drain; ++d) {
        if (--stage < 0) { stage = STAGES - 1; phase ^= 1; }
        mbar_wait_settle(&full[stage], phase, p.status, kDevTimeoutProducer);
      }
    }
  } else if (warp == 1 || warp == 2) {
    // ----------------------------------------------------------------- MMA
    if (elect_one()) {
      const int me = warp - 1;  // this thread's A tile
      const uint32_t op0 = smem_u32(smem) + me * C::A_BYTES;
      const uint32_t sf0 = smem_u32(smem + C::SF0);
      const uint32_t tsf0 = tmem + C::SF_BASE + me * C::SF_COLS;
      int stage = 0, nb = 0, i = 0;
      uint32_t phase = 0, tphase = 0;  // tphase: one bit per half
      bool ok = true;
      for (; ok; ++i) {
        const int ri = i % RING;
        if (!mbar_wait(&ufull[ri], (i / RING) & 1, p.status, kDevTimeoutMma, s_abort)) break;
        if (plan[ri].ncols == 0) break;
        const int m1 = plan[ri].m1, n = plan[ri].n, both = plan[ri].both, kb0 = plan[ri].kb0, kb1 = plan[ri].kb1;
        mbar_arrive(&uempty[ri]);
        const int nn = both ? 2 * n : n;  // columns of one accumulator
        const bool big = 2 * nn > C::HALF;
        const int b0 = big ? 0 : nb, b1 = big ? 1 : nb;
        for (int b = b0; b <= b1 && ok; ++b) {
          ok = mbar_wait(&tempty[b], ((tphase >> b) & 1) ^ 1, p.status, kDevTimeoutMma, s_abort);
          tphase ^= 1u << b;
        }
        if (!ok) break;
        const uint32_t d = tmem + b0 * C::HALF + me * nn;
        const bool mine = me == 0 || m1 >= 0;
        const uint32_t id0 = idesc_scaled<FP4>(nn);
        // One stage: scale atoms to TMEM, then its MMAs, all in order.
        auto issue = [&](int nkb, auto two_terms, uint32_t acc) {
          const uint32_t st = op0 + stage * C::OP_BYTES;
          const uint32_t sb = op0 - me * C::A_BYTES + stage * C::OP_BYTES + C::B_OFF;
          const uint32_t sf = sf0 + stage * C::SF_BYTES;
          const uint32_t ta = tsf0 + stage * (2 * C::SF_COLS), tb = ta + C::KB_STAGE * 4;
          const uint64_t da = umma_desc_sw128(st), db = umma_desc_sw128(sb), dl = umma_desc_sw128(sb + BN * 128);
#pragma unroll
          for (int h = 0; h < C::KB_STAGE; ++h) {
            if (h < nkb) {
              copy_scales(ta + h * 4, sf + h * 1024 + me * 512);
#pragma unroll
              for (int a = 0; a < C::ATOMS; ++a)
                copy_scales(tb + (h * C::ATOMS + a) * 4, sf + C::SFA_BYTES + (h * C::ATOMS + a) * 512);
            }
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {  // 32 bytes of a row each
            const int h = FP4 ? kk >> 1 : 0;
            if (h < nkb) {
              const uint32_t id = id0 | sf_id(FP4 ? (kk & 1) * 2 : kk);
              const uint32_t va = ta + h * 4, vb = tb + h * C::ATOMS * 4;
              mma_scaled<FP4>(d, da + 2 * kk, db + 2 * kk, id, va, vb, kk ? 1u : acc);
              if constexpr (decltype(two_terms)::value) mma_scaled<FP4>(d, da + 2 * kk, dl + 2 * kk, id, va, vb, 1u);
            }
          }
        };
        for (int kb = kb0; kb < kb1; kb += C::KB_STAGE) {
          if (!mbar_wait(&full[stage], phase, p.status, kDevTimeoutMma, s_abort)) { ok = false; break; }
          tc_fence_after();
          if (mine) {
            const uint32_t acc = kb > kb0;
            if (FP4 || both) issue(min(C::KB_STAGE, kb1 - kb), False{}, acc);
            else issue(1, True{}, acc);
          }
          mma_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        for (int b = b0; b <= b1; ++b) mma_commit(&tfull[b]);
        if (!big) nb ^= 1;
      }
      // Every MMA of both issuers ends before TMEM is freed, also after an abort.
      mma_commit(done_bar);
      mbar_wait_settle(done_bar, 0, p.status, kDevTimeoutMma);
    }
  } else if (C::RAW && warp >= EPI_WARP0 + C::EPI) {
    if constexpr (C::RAW) {
      // -------------------------------------------------------- rows (RAW only)
      // bf16: one token tile, rows 0 to ncols - 1 of every unit. Loads are issued
      // before the wait for the stage.
      const int me = (warp - EPI_WARP0 - C::EPI) % STAGES;      // this warp's stage
      const int row0 = (warp - EPI_WARP0 - C::EPI) / STAGES * 16;  // and its first bf16 row
      int done = 0;  // stages of earlier units
      bool ok = warp < EPI_WARP0 + C::EPI + C::PREP;
      for (int i = 0; ok; ++i) {
        const int ri = i % RING;
        if (!mbar_wait(&ufull[ri], (i / RING) & 1, p.status, kDevTimeoutProducer, s_abort)) break;
        const Unit e = plan[ri];
        if (e.ncols == 0) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&uempty[ri]);
        const int stages = (e.kb1 - e.kb0 + C::KB_STAGE - 1) / C::KB_STAGE;
        for (int j = (me + STAGES - done % STAGES) % STAGES; j < stages; j += STAGES) {
          const int kb = e.kb0 + j * C::KB_STAGE, stage = me;
          const uint32_t phase = (done + j) / STAGES & 1;
          uint8_t* sfb = smem + C::SF0 + stage * C::SF_BYTES + C::SFA_BYTES;
          if constexpr (FP4) {
            const uint32_t* words = static_cast<const uint32_t*>(p.raw) + static_cast<long long>(e.row0) * KB + kb;
            uint32_t v[C::KB_STAGE][BN / 32];
#pragma unroll
            for (int h = 0; h < C::KB_STAGE; ++h)
#pragma unroll
              for (int r = 0; r < BN / 32; ++r)
                v[h][r] = kb + h < e.kb1 && 32 * r + lane < e.ncols
                            ? __ldg(words + (32 * r + lane) * static_cast<long long>(KB) + h) : 0;
            if (!(ok = mbar_wait(&empty[stage], phase ^ 1, p.status, kDevTimeoutProducer, s_abort))) break;
#pragma unroll
            for (int h = 0; h < C::KB_STAGE; ++h)
#pragma unroll
              for (int r = 0; r < BN / 32; ++r)
                reinterpret_cast<uint32_t*>(sfb + h * C::ATOMS * 512)[lane * 4 + r] = v[h][r];
          } else {
            const int sub = lane & 7;  // 16 columns of the K block
            Cols c[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int r = row0 + 4 * t + (lane >> 3);
              c[t] = Cols{};
              if (r < e.ncols) {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.raw) +
                                                                  r * p.raw_stride + kb * 128 + sub * 16);
                c[t].a = __ldg(src);
                c[t].b = __ldg(src + 1);
              }
            }
            if (!(ok = mbar_wait(&empty[stage], phase ^ 1, p.status, kDevTimeoutProducer, s_abort))) break;
            __syncwarp();
            uint8_t* b = smem + stage * C::OP_BYTES + C::B_OFF;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              if (row0 + 4 * t < e.ncols) {  // warp-uniform
                const int r = row0 + 4 * t + (lane >> 3), lo = e.n + r;  // hi and lo side by side
                uint32_t hw[4], lw[4], word;
                split_cols(c[t], hw, lw, word);
                if (r < e.ncols) {
                  // n is a multiple of 8: both rows have the same place in the swizzle
                  const int chunk = (sub ^ (r & 7)) * 16;
                  *reinterpret_cast<uint4*>(b + r * 128 + chunk) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
                  *reinterpret_cast<uint4*>(b + lo * 128 + chunk) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
                  if (sub == 0) {
                    reinterpret_cast<uint32_t*>(sfb)[r * 4] = word;
                    reinterpret_cast<uint32_t*>(sfb)[(lo & 31) * 4 + (lo >> 5)] = word;
                  }
                }
              }
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
        }
        done += stages;
      }
    }
  } else if (warp >= EPI_WARP0) {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3;
    const int cg = (warp - EPI_WARP0) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    int nb = 0, i = 0;
    uint32_t tphase = 0;  // one bit per half
    bool ok = true;
    for (; ok; ++i) {
      const int ri = i % RING;
      if (!mbar_wait(&ufull[ri], (i / RING) & 1, p.status, kDevTimeoutEpilogue, s_abort)) break;
      const Unit e = plan[ri];
      if (e.ncols == 0) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&uempty[ri]);
      const int nn = e.both ? 2 * e.n : e.n;
      const bool big = 2 * nn > C::HALF;
      const int b0 = big ? 0 : nb, b1 = big ? 1 : nb;
      for (int b = b0; b <= b1 && ok; ++b) {
        ok = mbar_wait(&tfull[b], (tphase >> b) & 1, p.status, kDevTimeoutEpilogue, s_abort);
        tphase ^= 1u << b;
      }
      if (!ok) break;
      if (!big) nb ^= 1;
      tc_fence_after();
      const uint32_t d0 = tmem + lanes + b0 * C::HALF, d1 = d0 + nn;
      const bool two = e.m1 >= 0;
      // 8 columns from column c on of one accumulator, hi + lo
      auto load = [&](uint32_t d, int c, float* v) {
        tmem_ld8(d + c, v);
        if (!FP4 && e.both) {
          float l[CHUNK];
          tmem_ld8(d + e.n + c, l);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < CHUNK; ++j) v[j] += l[j];
        } else {
          tmem_ld_wait();
        }
      };
      auto column = [&](int j) { return (j * C::NUM_CG + cg) * CHUNK; };  // of this warp's j-th chunk
      // The accumulators are read into registers and given back before the
      // results are rounded and stored: a large unit's MMAs start behind
      // nothing but that read.
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0)
          for (int b = b0; b <= b1; ++b) mbar_arrive(&tempty[b]);
      };
      if constexpr (SWIGLU) {
        float h[C::CHUNKS * CHUNK];
#pragma unroll
        for (int j = 0; j < C::CHUNKS; ++j) {
          if (column(j) < e.ncols) {  // warp-uniform
            float g[CHUNK], up[CHUNK];
            load(d0, column(j), g);
            load(d1, column(j), up);
            // silu in fp32 with the fast exp and divide. __expf is off by 2 +
            // 1.173 |g| units in the last place, the divide by 2: relative error up
            // to (5 + 1.2 |g|) 2^-23 (29 units at g = -20, 101 at -80). Where 1 +
            // e^-g passes 2^126 (g below -87.3) the divide may give 0, of a silu
            // below 2^-119. All far below the 2^-9 that the split keeps.
#pragma unroll
            for (int t = 0; t < CHUNK; ++t) h[j * CHUNK + t] = __fdividef(g[t], 1.0f + __expf(-g[t])) * up[t];
          }
        }
        release();
        const int f0 = e.m0 + quad * 32;  // this warp's 32 features: one scale block
        uint8_t* sf = p.hsf + (static_cast<size_t>(e.tile) * (p.M / 128) + e.m0 / 128) * (C::ATOMS * 512) + quad;
        auto spot = [](int c) { return (c >> 7) * 512 + (c & 31) * 16 + ((c >> 5) & 3) * 4; };
#pragma unroll
        for (int j = 0; j < C::CHUNKS * CHUNK; j += 4) {
          const int c0 = column(j / CHUNK) + j % CHUNK;
          if (c0 < e.ncols) {
            uint32_t hi4, lo4, bytes = 0;
            float q[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint32_t ef = __reduce_max_sync(0xffffffffu, __float_as_uint(h[j + t]) & 0x7fffffffu) >> 23;
              const uint32_t byte = ef == 255 ? 255u : (ef > 7 ? ef - 7 : 0u);
              q[t] = h[j + t] * (ef == 255 ? 0.f : __uint_as_float((254u - byte) << 23));
              bytes |= byte << (8 * t);
            }
            // f16's 11 bits on the way to the two terms' 8 or 9
            split4(f16_pair(q[0], q[1]), f16_pair(q[2], q[3]), hi4, lo4);
            hi4 = transpose4(hi4, lane);
            lo4 = transpose4(lo4, lane);
            const int col = c0 + (lane & 3);
            if (col < e.ncols) {
              const size_t off = static_cast<size_t>(e.row0 + col) * p.M + f0 + (lane & ~3);
              *reinterpret_cast<uint32_t*>(p.hq + off) = hi4;
              *reinterpret_cast<uint32_t*>(p.hq + static_cast<size_t>(p.P) * p.M + off) = lo4;
              if (lane < 4) {
                const uint8_t byte = static_cast<uint8_t>(bytes >> (8 * lane));
                sf[spot(col)] = byte;
                if (e.both) sf[spot(col + e.n)] = byte;
              }
            }
          }
        }
      } else if (p.ksplit == 1) {
        uint32_t y2[2][C::CHUNKS * CHUNK / 2];  // bf16 pairs of tokens
#pragma unroll
        for (int j = 0; j < C::CHUNKS; ++j) {
          if (column(j) < e.ncols) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              if (a == 0 || two) {
                float v[CHUNK];
                load(a ? d1 : d0, column(j), v);
#pragma unroll
                for (int t = 0; t < CHUNK; t += 2) {
                  const __nv_bfloat162 w = __floats2bfloat162_rn(v[t], v[t + 1]);
                  y2[a][(j * CHUNK + t) / 2] = *reinterpret_cast<const uint32_t*>(&w);
                }
              }
            }
          }
        }
        release();
        const int f = quad * 32 + (lane & ~3);  // M is a multiple of 8: four features are in or out together
#pragma unroll
        for (int j = 0; j < C::CHUNKS * CHUNK; j += 4) {
          const int c0 = column(j / CHUNK) + j % CHUNK;
          if (c0 < e.ncols) {
            const int col = c0 + (lane & 3);
            __nv_bfloat16* y = p.y + static_cast<size_t>(e.row0 + col) * p.M + f;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              if (a == 0 || two) {
                const int m = a ? e.m1 : e.m0;
                const uint2 v = transpose4(y2[a][j / 2], y2[a][j / 2 + 1], lane);
                if (col < e.ncols && m + f < p.M) *reinterpret_cast<uint2*>(y + m) = v;
              }
            }
          }
        }
      } else {
        // This part's sums, fp32, into the (now unused) operand stages:
        // [column][256 features].
        float* part = reinterpret_cast<float*>(smem) + quad * 32 + lane;
        for (int c0 = cg * CHUNK; c0 < e.ncols; c0 += C::NUM_CG * CHUNK) {
          float v[CHUNK];
          for (int a = 0; a < (two ? 2 : 1); ++a) {
            load(a ? d1 : d0, c0, v);
#pragma unroll
            for (int j = 0; j < CHUNK; ++j)
              if (c0 + j < e.ncols) part[(c0 + j) * 2 * BM + a * BM] = v[j];
          }
        }
        release();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
  if constexpr (!SWIGLU) {
    if (p.ksplit > 1) {
      // The cluster's CTAs hold the parts of one tile. Each adds up its share
      // of the columns over all of them, in part order, from their shared
      // memory. Every thread of every CTA passes both barriers, also after an
      // abort (the sums are then meaningless and the status says so).
      cluster_sync();
      const Unit e = plan[0];  // the CTA's only unit
      const int m = 2 * (threadIdx.x & 127);
      if (e.m0 + m < p.M) {
        const float* mine = reinterpret_cast<const float*>(smem) + m;
        for (int c = e.part + p.ksplit * (threadIdx.x >> 7); c < e.ncols; c += p.ksplit * (THREADS / 128)) {
          float2 v[kMaxSplit];
#pragma unroll
          for (int s = 0; s < kMaxSplit; ++s)
            if (s < p.ksplit) v[s] = load_peer(mine + c * 2 * BM, s);
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int s = 0; s < kMaxSplit; ++s)
            if (s < p.ksplit) x += v[s].x, y += v[s].y;
          *reinterpret_cast<__nv_bfloat162*>(p.y + static_cast<size_t>(e.row0 + c) * p.M + e.m0 + m) =
              __floats2bfloat162_rn(x, y);
        }
      }
      cluster_sync();  // no CTA exits while another reads its shared memory
    }
  }
}

template <class C, bool SWIGLU>
cudaError_t prepare(int* dev) {
  static std::atomic<bool> attr[64];  // threads that come together set it twice
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return e;
  if (*dev < 0 || *dev >= 64) return cudaErrorInvalidDevice;
  if (!attr[*dev]) {
    e = cudaFuncSetAttribute(mx_gemm_kernel<C, SWIGLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    attr[*dev] = true;
  }
  return cudaSuccess;
}

template <class C>
cudaLaunchConfig_t config(bool chained, int grid, cudaStream_t s, cudaLaunchAttribute* at, int cluster) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = THREADS;
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cfg.attrs = at;
  if (chained && !C::RAW) {  // RAW: it is the call's first kernel
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = cluster;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  return cfg;
}

template <class C, bool SWIGLU>
cudaError_t launch(bool chained, const CUtensorMap& w0, const CUtensorMap& w1, const CUtensorMap& x,
                   const CUtensorMap& x32, const CUtensorMap& x8, const GemmArgs& a, int grid, cudaStream_t s) {
  int dev = 0;
  const cudaError_t e = prepare<C, SWIGLU>(&dev);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute at[2];
  const cudaLaunchConfig_t cfg = config<C>(chained, grid, s, at, a.ksplit);
  return cudaLaunchKernelEx(&cfg, mx_gemm_kernel<C, SWIGLU>, w0, w1, x, x32, x8, a);
}

// Clusters of `split` CTAs that run at the same time on the current device.
template <class C>
int resident_clusters(int split) {
  static std::atomic<int> cache[64][kMaxSplit + 1];
  int dev = 0;
  if (prepare<C, false>(&dev) != cudaSuccess) return 0;
  int n = cache[dev][split].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchAttribute at[2];
    cudaLaunchConfig_t cfg = config<C>(true, split, nullptr, at, split);
    if (cudaOccupancyMaxActiveClusters(&n, mx_gemm_kernel<C, false>, &cfg) != cudaSuccess) n = -1;
    cache[dev][split].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace

// The widest split that keeps four K blocks per part and runs in one wave.
int pick_ksplit(bool fp4, int tile, int units, int kblocks) {
  int best = 1;
  for (int s = 2; s <= kMaxSplit && s * 4 <= kblocks; ++s) {
    int n = 0;
    if (fp4) n = tile == 64 ? resident_clusters<Cfg<true, 64, 4, true>>(s) : resident_clusters<Cfg<true, 160, 4>>(s);
    else n = tile == 16 ? resident_clusters<Cfg<false, 16, 6, true>>(s)
             : tile == 32 ? resident_clusters<Cfg<false, 32, 5>>(s)
             : tile == 64 ? resident_clusters<Cfg<false, 64, 4>>(s)
             : tile == 128 ? resident_clusters<Cfg<false, 128, 3>>(s) : resident_clusters<Cfg<false, 160, 3>>(s);
    if (n >= units) best = s;
  }
  return best;
}

cudaError_t launch_gemm(bool chained, bool fp4, bool swiglu, const CUtensorMap& w0, const CUtensorMap& w1,
                        const CUtensorMap& x, const CUtensorMap& x32, const CUtensorMap& x8, const GemmArgs& a,
                        int tile, int grid, cudaStream_t s) {
  if (fp4) {
    switch (tile) {
      case 64: return launch<Cfg<true, 64, 4, true>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
      case 160: return launch<Cfg<true, 160, 4>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
      default: return cudaErrorInvalidValue;
    }
  }
  switch (tile) {
    case 16:  // single-group products of up to 16 rows only
      return swiglu ? cudaErrorInvalidValue : launch<Cfg<false, 16, 6, true>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
    case 32:
      if (a.raw) return launch<Cfg<false, 32, 5, true>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
      return swiglu ? launch<Cfg<false, 32, 5>, true>(chained, w0, w1, x, x32, x8, a, grid, s)
                    : launch<Cfg<false, 32, 5>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
    case 64:
      return swiglu ? launch<Cfg<false, 64, 4>, true>(chained, w0, w1, x, x32, x8, a, grid, s)
                    : launch<Cfg<false, 64, 4>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
    case 128:  // single-group products only
      return swiglu ? cudaErrorInvalidValue : launch<Cfg<false, 128, 3>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
    case 160:
      return swiglu ? launch<Cfg<false, 160, 3>, true>(chained, w0, w1, x, x32, x8, a, grid, s)
                    : launch<Cfg<false, 160, 3>, false>(chained, w0, w1, x, x32, x8, a, grid, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace mx
}  // namespace dsmoe
