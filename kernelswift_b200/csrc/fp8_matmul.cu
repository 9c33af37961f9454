// Dense block-scaled fp8 product
//   out[t, n] = addend[t, n] + sum_kb sx[t, kb] sw[n / 128, kb]
//                              sum_{k in block kb} xq[t, k] wq[n, k]
// with e4m3 operands xq [T, K] and wq [N, K] on the tcgen05 tensor cores.
//
// Two kernels, by where the scales are applied and which operand lies on the
// MMA's 128 rows (TMEM lanes):
//
// fp8_cols_kernel: a tile is 128 weight rows (lanes) x BN tokens (columns),
//   BN in {16, ..., 256}, so that a handful of tokens costs a handful of
//   columns. UE8M0 scales are applied by the tensor core (kind::mxf8f6f4,
//   block_scale): all k-blocks accumulate in one TMEM accumulator. fp32 scales
//   cannot be: each k-block's product goes to a TMEM buffer of its own and is
//   added to fp32 registers times sx * sw, which a warp brings to shared
//   memory per k-block (a column's factor is the same for all lanes). Tiles
//   too few for the SMs are split along K over a cluster of up to 8 CTAs,
//   whose fp32 partials are summed in rank order through distributed shared
//   memory: one launch, no workspace, a fixed order of summation.
//
// fp8_rows_kernel: fp32 scales and many tokens. A tile is 128 tokens (lanes) x
//   256 weight rows (columns): a thread's columns share one sw and its row one
//   sx, so the promotion needs a single factor per thread and k-block instead
//   of one per column (shared-memory reads that would compete with the MMA's
//   operand reads).
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "runtime.h"

namespace ksw {
namespace {

constexpr int kKB = 128;            // bytes (= columns) of a k-block
constexpr int kLanes = 128;         // rows of the MMA
constexpr int kABytes = kLanes * kKB;
constexpr int kSfSlots = 4;         // scale ring: quads of 4 k-blocks (UE8M0)
constexpr int kFacSlots = 8;        // scale ring: k-blocks (fp32)

constexpr int kStagedBytes = 4096;  // staged tokens of one epilogue group (two such buffers)

struct MatmulParams {
  const void* xs;  // activation scales, f32 or bytes
  int64_t xs_row, xs_blk;
  const void* ws;  // weight scales [ceil(N / 128), KB] dense
  void* out;
  int64_t ld_out;
  const void* add;  // may be null
  int64_t ld_add;
  int64_t T, N;
  int kb_total;            // k-blocks
  int t_tiles, n_tiles;
  int splits;              // CTAs of a cluster that share a tile
  int32_t* status;
  uint64_t wait_limit_ns;
};

// Tiles in groups of kGroupT token tiles, weight tiles slowest inside a
// group: the CTAs of a wave share few rows of both operands through L2.
constexpr int kGroupT = 8;
struct Tile {
  int t, n;
};
__device__ __forceinline__ Tile tile_at(int i, int t_tiles, int n_tiles) {
  const int per = kGroupT * n_tiles;
  const int g = i / per, r = i - g * per;
  const int wide = min(kGroupT, t_tiles - g * kGroupT);
  const int n = r / wide;
  return {g * kGroupT + (r - n * wide), n};
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
               "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-memory word of CTA `rank` at this CTA's address `addr`.
__device__ __forceinline__ float ld_peer(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// Waits for this thread's tensor-memory loads; the values read pass through
// the (empty) statements after it, so no use of them can move before it.
template <int N>
__device__ __forceinline__ void tmem_arrived(uint32_t (&v)[N]) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}

// The last phase of each stage of a TMA ring that issued `issued` boxes: waits
// until none is in flight (a kernel must not end before its copies).
__device__ __forceinline__ void drain_ring(uint64_t* full, int stages, uint32_t issued,
                                           uint64_t limit) {
  for (int s = 0; s < stages; ++s) {
    const uint32_t n = issued / stages + (uint32_t(s) < issued % stages ? 1u : 0u);
    if (n == 0) continue;
    volatile int no_abort = 0;
    mbar_wait_bounded(&full[s], (n - 1) & 1u, &no_abort, limit);
  }
}

// Four consecutive scale bytes 4q .. 4q + 3 of one row (bytes past KB are 0).
__device__ __forceinline__ uint32_t scale_word(const uint8_t* row, int64_t stride, int q, int kb,
                                               bool words) {
  if (words && 4 * q + 4 <= kb) return __ldg(reinterpret_cast<const uint32_t*>(row + 4 * q));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * q + i < kb) w |= uint32_t(__ldg(row + int64_t(4 * q + i) * stride)) << (8 * i);
  return w;
}

// ---------------------------------------------------------------------------
// fp8_cols_kernel
// ---------------------------------------------------------------------------
template <bool MX, int BN>
struct ColsCfg {
  static constexpr int kEpiWarps = BN >= 128 ? 8 : 4;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kCols = BN / (kEpiWarps / 4);  // columns per epilogue warp
  static constexpr int kCtas = BN <= 64 ? 2 : 1;      // CTAs per SM
  static constexpr int kBBytes = BN * kKB;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kSfb = (BN + 127) / 128;       // scale chunks of the tokens
  static constexpr int kRingBytes = MX ? kSfSlots * 512 * (1 + kSfb) : kFacSlots * BN * 4;
  static constexpr int kGroups = kEpiWarps / 4;       // epilogue groups of 128 lanes
  static constexpr size_t kFixed = 1024 + 512 + kRingBytes + size_t(kGroups) * 2 * kStagedBytes;
  static constexpr int kStages = int(((kCtas == 2 ? 112 : 224) * 1024 - kFixed) / kStageBytes);
  static constexpr size_t kSmem = kFixed + size_t(kStages) * kStageBytes;
  // TMEM: accumulators (UE8M0) or per-k-block buffers (fp32), then scale slots
  static constexpr int kBufs = MX ? (BN == 256 ? 1 : 2) : (BN == 256 ? 2 : 4);
  static constexpr int kSfCol0 = kBufs * BN;
  static constexpr int kSfCols = 4 * (1 + kSfb);
  static constexpr int kUsed = kSfCol0 + (MX ? kSfSlots * kSfCols : 0);
  static constexpr int kTmem = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(kUsed <= 512 && kTmem * kCtas <= 512, "TMEM columns");
  static_assert(size_t(kStages) * kStageBytes >= size_t(BN) * kLanes * 4,
                "the partial tile reuses the stages");
  static_assert(8 * (2 * kStages + 2 * kFacSlots + 2 * 4 + 1) + 8 <= 512, "barriers");
};

template <bool MX, int BN, typename TOUT>
__global__ void __launch_bounds__(ColsCfg<MX, BN>::kThreads, ColsCfg<MX, BN>::kCtas)
    fp8_cols_kernel(const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmX, const MatmulParams p) {
  using C = ColsCfg<MX, BN>;
  constexpr int STAGES = C::kStages;
  constexpr int NB = C::kBufs;
  constexpr int COLS = C::kCols;
  constexpr int SLOTS = MX ? kSfSlots : kFacSlots;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * kABytes;
  uint8_t* sRing = sB + STAGES * C::kBBytes;
  uint8_t* sOut = sRing + C::kRingBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + C::kGroups * 2 * kStagedBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* sfull = empty + STAGES;
  uint64_t* sempty = sfull + SLOTS;
  uint64_t* tfull = sempty + SLOTS;
  uint64_t* tempty = tfull + NB;
  uint64_t* final_bar = tempty + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(final_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&sfull[s], 32);
      mbar_init(&sempty[s], MX ? 1 : C::kEpiWarps);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], C::kEpiWarps);
    }
    mbar_init(final_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  const uint64_t limit = p.wait_limit_ns;
  const int tiles = p.t_tiles * p.n_tiles;
  // a cluster's CTAs share a tile: CTA `part` takes k-blocks [kb0, kb1)
  const int part = int(blockIdx.x) % p.splits;
  const int first = int(blockIdx.x) / p.splits, step = int(gridDim.x) / p.splits;
  const int kb0 = int(int64_t(p.kb_total) * part / p.splits);
  const int kb1 = int(int64_t(p.kb_total) * (part + 1) / p.splits);

  float acc[COLS];  // the epilogue warps' tile columns
#pragma unroll
  for (int j = 0; j < COLS; ++j) acc[j] = 0.0f;
  bool epi_ok = true;

  // 16-byte stores when every output row starts on such a boundary
  constexpr int kVec = 16 / int(sizeof(TOUT));
  const bool vec = p.ld_out % kVec == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;

  // Writes the tile's columns (tokens) col0 .. col0 + COLS of this epilogue
  // group's 128 lanes (weight rows, neighbours in the output). A lane holds
  // one output column of every token; tokens go through shared memory, a few
  // at a time, so that a warp stores whole 128-byte lines.
  auto store_tile = [&](const Tile& tile, int col0, int row, int group) {
    const int64_t n0 = int64_t(tile.n) * kLanes;
    const int64_t t0 = int64_t(tile.t) * BN + col0;
    const int64_t live = min(int64_t(COLS), p.T - t0);
    const bool in = n0 + row < p.N;
    TOUT* out = static_cast<TOUT*>(p.out) + t0 * p.ld_out + n0;
    if (p.add != nullptr) {
      const TOUT* add = static_cast<const TOUT*>(p.add) + t0 * p.ld_add + n0 + row;
#pragma unroll
      for (int j = 0; j < COLS; ++j) {
        if (in && j < live) acc[j] += to_f32(*add);
        add += p.ld_add;
      }
    }
    if (!vec) {
      out += row;
#pragma unroll
      for (int j = 0; j < COLS; ++j) {
        if (in && j < live) *out = from_f32<TOUT>(acc[j]);
        out += p.ld_out;
      }
      return;
    }
    constexpr int TOK = kStagedBytes / (kLanes * int(sizeof(TOUT)));  // tokens per buffer
    constexpr int SEGS = kLanes / kVec;                               // vectors per token
    TOUT* staged = reinterpret_cast<TOUT*>(sOut + group * 2 * kStagedBytes);
#pragma unroll
    for (int c = 0; c < COLS; c += TOK) {
      if (c >= live) break;
      TOUT* buf = staged + ((c / TOK) & 1) * (TOK * kLanes);
#pragma unroll
      for (int j = 0; j < TOK; ++j) buf[j * kLanes + row] = from_f32<TOUT>(acc[c + j]);
      // the buffer's readers of two chunks ago passed the last chunk's barrier
      asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
#pragma unroll
      for (int i = 0; i < TOK * SEGS / 128; ++i) {
        const int v = row + 128 * i;
        const int j = v / SEGS, seg = v % SEGS;
        const uint4 w = reinterpret_cast<const uint4*>(buf)[v];
        if (c + j >= live) continue;
        TOUT* dst = out + (c + j) * p.ld_out + seg * kVec;
        const int64_t left = p.N - n0 - seg * kVec;
        if (left >= kVec) {
          *reinterpret_cast<uint4*>(dst) = w;
        } else {
          const TOUT* e = reinterpret_cast<const TOUT*>(&w);
#pragma unroll
          for (int k = 0; k < kVec; ++k)
            if (k < left) dst[k] = e[k];
        }
      }
    }
    // the next tile starts with buffer 0 again
    asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
  };

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer ----------------
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    int stage = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag, limit)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
        tma_load_2d(sA + stage * kABytes, &tmW, kb * kKB, tile.n * kLanes, &full[stage]);
        tma_load_2d(sB + stage * C::kBBytes, &tmX, kb * kKB, tile.t * BN, &full[stage]);
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    drain_ring(full, STAGES, issued, limit);
  } else if (warp == 1 && lane == 0) {
    // ---------------- MMA issuer ----------------
    int stage = 0, buf = 0, slot = 0;
    uint32_t phase = 0, bphase = 0, sphase = 0;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      if constexpr (MX) {
        if (!mbar_wait_bounded(&tempty[buf], bphase ^ 1u, abort_flag, limit)) break;
        tc_fence_after();
      }
      for (int kb = kb0; kb < kb1; ++kb) {
        if constexpr (MX) {
          if (kb == kb0 || (kb & 3) == 0) {
            if (!mbar_wait_bounded(&sfull[slot], sphase, abort_flag, limit)) {
              ok = false;
              break;
            }
            tc_fence_after();
            // a slot's TMEM columns are rewritten only after sempty, i.e. after
            // the MMAs that read them completed
            const uint32_t sf = tmem_base + uint32_t(C::kSfCol0 + slot * C::kSfCols);
            const uint32_t src = smem_u32(sRing + slot * 512 * (1 + C::kSfb));
#pragma unroll
            for (int c = 0; c < 1 + C::kSfb; ++c)
              tc_cp_sf(sf + 4 * c, make_sf_desc(src + 512 * c));
          }
        } else {
          if (!mbar_wait_bounded(&tempty[buf], bphase ^ 1u, abort_flag, limit)) {
            ok = false;
            break;
          }
        }
        if (!mbar_wait_bounded(&full[stage], phase, abort_flag, limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + uint32_t(buf * BN);
        const uint32_t a0 = smem_u32(sA + stage * kABytes);
        const uint32_t b0 = smem_u32(sB + stage * C::kBBytes);
        if constexpr (MX) {
          const uint32_t sf = tmem_base + uint32_t(C::kSfCol0 + slot * C::kSfCols);
          const uint32_t idesc = idesc_sf_ids(make_idesc_mx(kLanes, BN), uint32_t(kb & 3));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_mx(d, make_sw128_desc(a0 + kk * 32), make_sw128_desc(b0 + kk * 32), idesc, sf,
                      sf + 4, (kb > kb0 || kk > 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
          if (kb + 1 == kb1 || ((kb + 1) & 3) == 0) {
            tc_commit(&sempty[slot]);
            if (++slot == SLOTS) {
              slot = 0;
              sphase ^= 1u;
            }
          }
        } else {
          constexpr uint32_t idesc = make_idesc(1u, 0u, kLanes, BN);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma<kKindF8>(d, make_sw128_desc(a0 + kk * 32), make_sw128_desc(b0 + kk * 32),
                            idesc, kk > 0 ? 1u : 0u);
          tc_commit(&empty[stage]);
          tc_commit(&tfull[buf]);
          if (++buf == NB) {
            buf = 0;
            bphase ^= 1u;
          }
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      if constexpr (MX) {
        tc_commit(&tfull[buf]);
        if (++buf == NB) {
          buf = 0;
          bphase ^= 1u;
        }
      }
    }
    tc_commit(final_bar);
    volatile int no_abort = 0;
    mbar_wait_bounded(final_bar, 0, &no_abort, limit);
  } else if (warp == 2) {
    // ---------------- scales ----------------
    int slot = 0;
    uint32_t sphase = 0;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      if constexpr (MX) {
        const uint8_t* xs = static_cast<const uint8_t*>(p.xs);
        const uint8_t* ws = static_cast<const uint8_t*>(p.ws) + int64_t(tile.n) * p.kb_total;
        const bool words = p.xs_blk == 1 && p.xs_row % 4 == 0 &&
                           (reinterpret_cast<uintptr_t>(xs) & 3) == 0;
        for (int q = kb0 / 4; 4 * q < kb1; ++q) {
          // loads first, so that they are under way while the slot drains
          const uint32_t w = scale_word(ws, 1, q, p.kb_total, false);
          uint32_t v[C::kSfb][4];
#pragma unroll
          for (int c = 0; c < C::kSfb; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int64_t t = int64_t(tile.t) * BN + 128 * c + 32 * r + lane;
              const bool in = 128 * c + 32 * r < BN && t < p.T;
              v[c][r] = in ? scale_word(xs + t * p.xs_row, p.xs_blk, q, p.kb_total, words) : 0u;
            }
          ok = mbar_wait_bounded(&sempty[slot], sphase ^ 1u, abort_flag, limit);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint4* dst = reinterpret_cast<uint4*>(sRing + slot * 512 * (1 + C::kSfb));
          dst[lane] = make_uint4(w, w, w, w);
#pragma unroll
          for (int c = 0; c < C::kSfb; ++c)
            dst[32 * (1 + c) + lane] = make_uint4(v[c][0], v[c][1], v[c][2], v[c][3]);
          // the copies to tensor memory read it through the async proxy
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(&sfull[slot]);
          if (++slot == SLOTS) {
            slot = 0;
            sphase ^= 1u;
          }
        }
      } else {
        const float* xs = static_cast<const float*>(p.xs);
        const float* ws = static_cast<const float*>(p.ws) + int64_t(tile.n) * p.kb_total;
        constexpr int R = (BN + 31) / 32;
        for (int kb = kb0; kb < kb1; ++kb) {
          const float w = __ldg(ws + kb);
          float v[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int64_t t = int64_t(tile.t) * BN + 32 * r + lane;
            v[r] = t < p.T && 32 * r + lane < BN ? __ldg(xs + t * p.xs_row + kb * p.xs_blk) : 0.0f;
          }
          ok = mbar_wait_bounded(&sempty[slot], sphase ^ 1u, abort_flag, limit);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          float* dst = reinterpret_cast<float*>(sRing) + slot * BN;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (32 * r + lane < BN) dst[32 * r + lane] = v[r] * w;
          mbar_arrive(&sfull[slot]);
          if (++slot == SLOTS) {
            slot = 0;
            sphase ^= 1u;
          }
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------- promotion and epilogue ----------------
    const int row = (warp & 3) * 32 + lane;
    const int col0 = ((warp - 4) >> 2) * COLS;
    const uint32_t lane_base = tmem_base + (uint32_t((warp & 3) * 32) << 16) + uint32_t(col0);
    int buf = 0, slot = 0;
    uint32_t bphase = 0, sphase = 0;
    constexpr int BATCH = COLS >= 32 ? 32 : 16;
    for (int i = first; epi_ok && i < tiles; i += step) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      if constexpr (MX) {
        bool ok = mbar_wait_bounded(&tfull[buf], bphase, abort_flag, limit);
        epi_ok = __all_sync(0xffffffffu, ok);
        if (!epi_ok) break;
        tc_fence_after();
        const uint32_t base = lane_base + uint32_t(buf * BN);
        uint32_t v[COLS];
#pragma unroll
        for (int c = 0; c < COLS; c += BATCH) {
          if constexpr (BATCH == 32)
            tmem_ld32(base + c, *reinterpret_cast<uint32_t(*)[32]>(&v[c]));
          else
            tmem_ld16(base + c, *reinterpret_cast<uint32_t(*)[16]>(&v[c]));
        }
        tmem_arrived(v);
#pragma unroll
        for (int j = 0; j < COLS; ++j) acc[j] = __uint_as_float(v[j]);
        // the tile is in registers: the next one's MMAs may start
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[buf]);
        if (++buf == NB) {
          buf = 0;
          bphase ^= 1u;
        }
      } else {
#pragma unroll
        for (int j = 0; j < COLS; ++j) acc[j] = 0.0f;
        for (int kb = kb0; kb < kb1; ++kb) {
          bool ok = mbar_wait_bounded(&sfull[slot], sphase, abort_flag, limit) &&
                    mbar_wait_bounded(&tfull[buf], bphase, abort_flag, limit);
          epi_ok = __all_sync(0xffffffffu, ok);
          if (!epi_ok) break;
          tc_fence_after();
          const uint32_t base = lane_base + uint32_t(buf * BN);
          const float4* fac =
              reinterpret_cast<const float4*>(sRing) + (slot * BN + col0) / 4;
#pragma unroll
          for (int c = 0; c < COLS; c += BATCH) {
            uint32_t v[BATCH];
            if constexpr (BATCH == 32)
              tmem_ld32(base + c, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
            else
              tmem_ld16(base + c, *reinterpret_cast<uint32_t(*)[16]>(&v[0]));
            // the factors are read after it, so no product can move before it
            tmem_ld_wait();
            if (c + BATCH >= COLS) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&tempty[buf]);
            }
#pragma unroll
            for (int j = 0; j < BATCH; j += 4) {
              const float4 f = fac[(c + j) / 4];
              acc[c + j] = fmaf(f.x, __uint_as_float(v[j]), acc[c + j]);
              acc[c + j + 1] = fmaf(f.y, __uint_as_float(v[j + 1]), acc[c + j + 1]);
              acc[c + j + 2] = fmaf(f.z, __uint_as_float(v[j + 2]), acc[c + j + 2]);
              acc[c + j + 3] = fmaf(f.w, __uint_as_float(v[j + 3]), acc[c + j + 3]);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sempty[slot]);
          if (++buf == NB) {
            buf = 0;
            bphase ^= 1u;
          }
          if (++slot == SLOTS) {
            slot = 0;
            sphase ^= 1u;
          }
        }
        if (!epi_ok) break;
      }
      if (p.splits == 1) {
        store_tile(tile, col0, row, (warp - 4) >> 2);
      } else {
        // every MMA of this CTA's only tile has completed, so the stages are
        // free; [token][weight row], a warp writes 32 neighbouring words
        float* part_tile = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int j = 0; j < COLS; ++j) part_tile[(col0 + j) * kLanes + row] = acc[j];
      }
    }
  }

  __syncwarp();
  __syncthreads();
  if (p.splits > 1) {
    cluster_sync();
    // CTA r sums tokens r, r + splits, ... over the cluster, in rank order
    const Tile tile = tile_at(first, p.t_tiles, p.n_tiles);
    const int64_t n = int64_t(tile.n) * kLanes + (threadIdx.x & 127);
    const uint32_t base = smem_u32(smem) + 4u * (threadIdx.x & 127);
    if (!*abort_flag) {
      for (int j = int(threadIdx.x >> 7) * p.splits + part; j < BN;
           j += int(blockDim.x >> 7) * p.splits) {
        const int64_t t = int64_t(tile.t) * BN + j;
        if (t >= p.T) break;
        float v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          v[r] = r < p.splits ? ld_peer(base + uint32_t(j * kLanes * 4), uint32_t(r)) : 0.0f;
        float sum = v[0];
#pragma unroll
        for (int r = 1; r < 8; ++r) sum += v[r];
        if (n < p.N) {
          if (p.add != nullptr)
            sum += to_f32(static_cast<const TOUT*>(p.add)[t * p.ld_add + n]);
          static_cast<TOUT*>(p.out)[t * p.ld_out + n] = from_f32<TOUT>(sum);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its partial
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmem);
  }
  if (threadIdx.x == 0 && *abort_flag) report_status(p.status, MOE_ERR_TIMEOUT);
}

// ---------------------------------------------------------------------------
// fp8_rows_kernel: fp32 scales, 128 tokens x 256 weight rows per tile
// ---------------------------------------------------------------------------
struct RowsCfg {
  static constexpr int kBN = 256;
  static constexpr int kEpiWarps = 16;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kCols = kBN / (kEpiWarps / 4);  // 64
  static constexpr int kBBytes = kBN * kKB;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 4;
  static constexpr size_t kSmem = 1024 + 256 + size_t(kStages) * kStageBytes;
  static constexpr int kBufs = 2;
  // The block launches at kLaunchRegs registers per thread; the control
  // warpgroup gives registers back and the 16 epilogue warps take them, for 64
  // sums and a batch of 32 partials each. The split adds up to the launch's
  // total, which the host checks against the compiled kernel.
  static constexpr int kLaunchRegs = 96, kCtrlRegs = 32, kEpiRegs = 112;
  static_assert(128 * kCtrlRegs + 32 * kEpiWarps * kEpiRegs == kThreads * kLaunchRegs,
                "setmaxnreg split");
};

// Transposes 4 x 4 vectors among the lanes of a quad: lane i's vector c
// becomes lane c's vector i (its own inverse).
__device__ __forceinline__ uint4 shfl_xor4(const uint4& v, int m) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m),
                    __shfl_xor_sync(0xffffffffu, v.z, m), __shfl_xor_sync(0xffffffffu, v.w, m));
}
__device__ __forceinline__ uint4 pick(bool b, const uint4& x, const uint4& y) {
  return make_uint4(b ? x.x : y.x, b ? x.y : y.y, b ? x.z : y.z, b ? x.w : y.w);
}
__device__ __forceinline__ void swap_pair(uint4& lo, uint4& hi, bool up, int m) {
  const uint4 got = shfl_xor4(pick(up, lo, hi), m);
  lo = pick(up, got, lo);
  hi = pick(up, hi, got);
}
__device__ __forceinline__ void quad_transpose(uint4 (&v)[4], int lane) {
  swap_pair(v[0], v[1], lane & 1, 1);
  swap_pair(v[2], v[3], lane & 1, 1);
  swap_pair(v[0], v[2], lane & 2, 2);
  swap_pair(v[1], v[3], lane & 2, 2);
}

// 16 bytes of the output's type to and from fp32.
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* x) {
  if constexpr (std::is_same<T, float>::value)
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                      __float_as_uint(x[3]));
  else
    return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                      pack2<T>(x[6], x[7]));
}

template <typename TOUT>
__global__ void __launch_bounds__(RowsCfg::kThreads, 1)
    fp8_rows_kernel(const __grid_constant__ CUtensorMap tmX,
                    const __grid_constant__ CUtensorMap tmW, const MatmulParams p) {
  using C = RowsCfg;
  constexpr int STAGES = C::kStages;
  constexpr int NB = C::kBufs;
  constexpr int COLS = C::kCols;
  constexpr int BATCH = 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + STAGES * C::kBBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + NB;
  uint64_t* final_bar = tempty + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(final_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], C::kEpiWarps);
    }
    mbar_init(final_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();
  const uint64_t limit = p.wait_limit_ns;
  const int tiles = p.t_tiles * p.n_tiles;
  const int kbs = p.kb_total;

  if (warp < 4) setmaxnreg_dec<C::kCtrlRegs>();
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
    int stage = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < tiles; i += gridDim.x) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      for (int kb = 0; kb < kbs; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag, limit)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
        tma_load_2d(sA + stage * kABytes, &tmX, kb * kKB, tile.t * kLanes, &full[stage]);
        tma_load_2d(sB + stage * C::kBBytes, &tmW, kb * kKB, tile.n * C::kBN, &full[stage]);
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    drain_ring(full, STAGES, issued, limit);
  } else if (warp == 1 && lane == 0) {
    int stage = 0, buf = 0;
    uint32_t phase = 0, bphase = 0;
    bool ok = true;
    constexpr uint32_t idesc = make_idesc(1u, 0u, kLanes, C::kBN);
    for (int i = blockIdx.x; ok && i < tiles; i += gridDim.x) {
      for (int kb = 0; kb < kbs; ++kb) {
        if (!mbar_wait_bounded(&tempty[buf], bphase ^ 1u, abort_flag, limit) ||
            !mbar_wait_bounded(&full[stage], phase, abort_flag, limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + uint32_t(buf * C::kBN);
        const uint32_t a0 = smem_u32(sA + stage * kABytes);
        const uint32_t b0 = smem_u32(sB + stage * C::kBBytes);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          tc_mma<kKindF8>(d, make_sw128_desc(a0 + kk * 32), make_sw128_desc(b0 + kk * 32), idesc,
                          kk > 0 ? 1u : 0u);
        tc_commit(&empty[stage]);
        tc_commit(&tfull[buf]);
        if (++buf == NB) {
          buf = 0;
          bphase ^= 1u;
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    tc_commit(final_bar);
    volatile int no_abort = 0;
    mbar_wait_bounded(final_bar, 0, &no_abort, limit);
  } else if (warp >= 4) {
    setmaxnreg_inc<C::kEpiRegs>();
    const int row = (warp & 3) * 32 + lane;
    const int col0 = ((warp - 4) >> 2) * COLS;
    const uint32_t lane_base = tmem_base + (uint32_t((warp & 3) * 32) << 16) + uint32_t(col0);
    const float* xs = static_cast<const float*>(p.xs);
    const float* ws = static_cast<const float*>(p.ws);
    const int64_t w_blocks = (p.N + 127) / 128;
    // 16-byte stores when every output row starts on such a boundary
    constexpr int kVec = 16 / int(sizeof(TOUT));
    const bool vec = p.ld_out % kVec == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
    const bool add_vec = p.ld_add % kVec == 0 && (reinterpret_cast<uintptr_t>(p.add) & 15) == 0;
    int buf = 0;
    uint32_t bphase = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < tiles; i += gridDim.x) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      const int64_t t = int64_t(tile.t) * kLanes + row;
      const int64_t n0 = int64_t(tile.n) * C::kBN + col0;
      const bool live = t < p.T;
      const int64_t wb = min(n0 / 128, w_blocks - 1);  // columns past N have no scale
      const float* sx = xs + (live ? t * p.xs_row : 0);
      const float* sw = ws + wb * kbs;
      float acc[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[j] = 0.0f;
      // the next k-block's scales are on their way while this one is added
      float sx_n = __ldg(sx), sw_n = __ldg(sw);
      for (int kb = 0; kb < kbs; ++kb) {
        float s = sx_n * sw_n;
        if (kb + 1 < kbs) {
          sx_n = __ldg(sx + (kb + 1) * p.xs_blk);
          sw_n = __ldg(sw + kb + 1);
        }
        ok = mbar_wait_bounded(&tfull[buf], bphase, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t base = lane_base + uint32_t(buf * C::kBN);
#pragma unroll
        for (int c = 0; c < COLS; c += BATCH) {
          uint32_t v[BATCH];
          tmem_ld32(base + c, v);
          tmem_ld_wait();
          asm volatile("" : "+f"(s));  // no product can move before the wait
          if (c + BATCH >= COLS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[buf]);
          }
#pragma unroll
          for (int j = 0; j < BATCH; ++j)
            acc[c + j] = fmaf(s, __uint_as_float(v[j]), acc[c + j]);
        }
        if (++buf == NB) {
          buf = 0;
          bphase ^= 1u;
        }
      }
      if (!ok) continue;
      TOUT* out = static_cast<TOUT*>(p.out) + n0;
      const TOUT* add = static_cast<const TOUT*>(p.add) + n0;
      const int cols = int(min(int64_t(COLS), max(int64_t(0), p.N - n0)));
      if (vec && cols == COLS && (p.add == nullptr || add_vec)) {
        // a quad of lanes trades vectors so that it stores 64 bytes of one
        // row at a time (and reads the addend so)
        const int64_t t4 = t - (lane & 3);
        const int mine = (lane & 3) * kVec;
#pragma unroll
        for (int j = 0; j < COLS; j += 4 * kVec) {
          uint4 v[4];
          if (p.add != nullptr) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              v[r] = t4 + r < p.T ? *reinterpret_cast<const uint4*>(add + (t4 + r) * p.ld_add +
                                                                    j + mine)
                                  : make_uint4(0, 0, 0, 0);
            quad_transpose(v, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const TOUT* e = reinterpret_cast<const TOUT*>(&v[r]);
#pragma unroll
              for (int k = 0; k < kVec; ++k) acc[j + r * kVec + k] += to_f32(e[k]);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = pack16<TOUT>(&acc[j + r * kVec]);
          quad_transpose(v, lane);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t4 + r < p.T)
              *reinterpret_cast<uint4*>(out + (t4 + r) * p.ld_out + j + mine) = v[r];
        }
      } else if (live) {
        out += t * p.ld_out;
        add += t * p.ld_add;
#pragma unroll
        for (int j = 0; j < COLS; ++j)
          if (j < cols) {
            if (p.add != nullptr) acc[j] += to_f32(add[j]);
            out[j] = from_f32<TOUT>(acc[j]);
          }
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) report_status(p.status, MOE_ERR_TIMEOUT);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Plan {
  int rows;    // 1: fp8_rows_kernel
  int bn;      // columns per tile (tokens; weight rows for fp8_rows_kernel)
  int splits;  // CTAs per cluster along K
  int ctas;
};

Plan plan_matmul(int64_t T, int64_t N, int64_t K, bool mx, int sms) {
  const int64_t kbs = ceil_div(K, kKB);
  Plan best = {0, 16, 1, 1};
  if (!mx && T > 128) {
    const int64_t tiles = ceil_div(T, kLanes) * ceil_div(N, 256);
    return {1, 256, 1, int(std::min<int64_t>(tiles, sms))};
  }
  double best_cost = 1e300;
  for (int bn : {16, 32, 64, 128, 256}) {
    if (bn == 256 && !mx) continue;
    if (bn > 16 && bn / 2 >= T) continue;  // the half would hold every token
    const int64_t tiles = ceil_div(T, bn) * ceil_div(N, kLanes);
    for (int s = 1; s <= 8 && s <= kbs; ++s) {
      const int occ = bn <= 64 ? 2 : 1;
      if (s > 1 && tiles * s > int64_t(sms) * occ) break;
      // cycles: k-blocks one after another on an SM, each the MMA's or, when
      // longer, its share of the bytes an SM takes in; then a tile's epilogue
      const double per_kb = std::max(2.0 * bn, (kABytes + bn * kKB) / 56.0);
      const double per_tile = 400 + 4.0 * bn;
      const double waves = double(ceil_div(tiles * s, sms));
      const double cost = waves * (double(ceil_div(kbs, s)) * per_kb + per_tile) +
                          (s > 1 ? 1200 + 2.0 * bn : 0);
      if (cost < best_cost) {
        best_cost = cost;
        best = {0, bn, s,
                int(s > 1 ? tiles * s : std::min<int64_t>(tiles, int64_t(sms) * occ))};
      }
    }
  }
  return best;
}

template <typename Kern>
int set_smem_once(Kern kern, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  KSW_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? (uint64_t(1) << dev) : 0;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return MOE_OK;
  KSW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
  done.fetch_or(bit, std::memory_order_acq_rel);
  return MOE_OK;
}

template <typename Kern>
int launch_clusters(Kern kern, int grid, int threads, size_t smem, int cluster, cudaStream_t s,
                    const CUtensorMap& a, const CUtensorMap& b, const MatmulParams& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = unsigned(cluster);
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = unsigned(n);
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, b, p), "cudaLaunchKernelEx");
}

template <bool MX, int BN, typename TOUT>
int launch_cols(const Plan& plan, const CUtensorMap& w, const CUtensorMap& x,
                const MatmulParams& p, cudaStream_t s) {
  using C = ColsCfg<MX, BN>;
  static std::atomic<uint64_t> done{0};
  int st = set_smem_once(fp8_cols_kernel<MX, BN, TOUT>, C::kSmem, done);
  if (st != MOE_OK) return st;
  return launch_clusters(fp8_cols_kernel<MX, BN, TOUT>, plan.ctas, C::kThreads, C::kSmem,
                         plan.splits, s, w, x, p);
}

template <bool MX, typename TOUT>
int dispatch_cols(const Plan& plan, const CUtensorMap& w, const CUtensorMap& x,
                  const MatmulParams& p, cudaStream_t s) {
  switch (plan.bn) {
    case 16: return launch_cols<MX, 16, TOUT>(plan, w, x, p, s);
    case 32: return launch_cols<MX, 32, TOUT>(plan, w, x, p, s);
    case 64: return launch_cols<MX, 64, TOUT>(plan, w, x, p, s);
    case 128: return launch_cols<MX, 128, TOUT>(plan, w, x, p, s);
    default: break;
  }
  if constexpr (MX) return launch_cols<MX, 256, TOUT>(plan, w, x, p, s);
  return fail(MOE_ERR_UNSUPPORTED, "fp8_matmul: no such tile");
}

template <typename TOUT>
int run_matmul(const Plan& plan, bool mx, const CUtensorMap& w, const CUtensorMap& x,
               const MatmulParams& p, cudaStream_t s) {
  if (plan.rows) {
    static std::atomic<uint64_t> done{0};
    int st = set_smem_once(fp8_rows_kernel<TOUT>, RowsCfg::kSmem, done);
    if (st != MOE_OK) return st;
    // a register split that the launch cannot cover would never return
    static const int regs = [] {
      cudaFuncAttributes attr;
      return cudaFuncGetAttributes(&attr, fp8_rows_kernel<TOUT>) == cudaSuccess ? attr.numRegs
                                                                                : -1;
    }();
    KSW_REQUIRE(regs == RowsCfg::kLaunchRegs, MOE_ERR_UNSUPPORTED,
                "fp8_matmul: compiled register count does not match the setmaxnreg split");
    return launch_clusters(fp8_rows_kernel<TOUT>, plan.ctas, RowsCfg::kThreads, RowsCfg::kSmem, 1,
                           s, x, w, p);
  }
  return mx ? dispatch_cols<true, TOUT>(plan, w, x, p, s)
            : dispatch_cols<false, TOUT>(plan, w, x, p, s);
}

int check_sizes(int64_t T, int64_t N, int64_t K, int scale_format) {
  KSW_REQUIRE(T >= 0 && N >= 1 && K >= 1, MOE_ERR_INVALID_ARG, "fp8_matmul: bad sizes");
  KSW_REQUIRE(T < (int64_t(1) << 31) - 256 && N < (int64_t(1) << 31) - 256 &&
                  K < (int64_t(1) << 31) - 256,
              MOE_ERR_UNSUPPORTED, "fp8_matmul: sizes beyond 2^31");
  KSW_REQUIRE(ceil_div(T, 16) * ceil_div(N, 128) < (int64_t(1) << 27), MOE_ERR_UNSUPPORTED,
              "fp8_matmul: too many tiles");
  KSW_REQUIRE(scale_format == 0 || scale_format == 1, MOE_ERR_INVALID_ARG,
              "fp8_matmul: scale_format must be 0 (fp32) or 1 (UE8M0)");
  return MOE_OK;
}

}  // namespace
}  // namespace ksw

extern "C" int moe_fp8_matmul_plan(int64_t num_rows, int64_t out_cols, int64_t inner,
                                   int scale_format, int32_t* info) {
  using namespace ksw;
  int st = check_sizes(num_rows, out_cols, inner, scale_format);
  if (st != MOE_OK) return st;
  KSW_REQUIRE(info != nullptr, MOE_ERR_INVALID_ARG, "fp8_matmul_plan: null pointer");
  const Plan plan = plan_matmul(num_rows, out_cols, inner, scale_format == 1, 148);
  info[0] = plan.rows;
  info[1] = plan.bn;
  info[2] = plan.splits;
  info[3] = num_rows == 0 ? 0 : plan.ctas;
  return MOE_OK;
}

extern "C" int moe_fp8_matmul(const void* x, int64_t ld_x, const void* x_scale,
                              int64_t xs_row_stride, int64_t xs_block_stride, const void* w,
                              int64_t ld_w, const void* w_scale, int scale_format,
                              int64_t num_rows, int64_t out_cols, int64_t inner,
                              const void* addend, int64_t ld_addend, void* out, int64_t ld_out,
                              int out_dtype, int32_t* status, void* stream) {
  using namespace ksw;
  int st = check_sizes(num_rows, out_cols, inner, scale_format);
  if (st != MOE_OK) return st;
  KSW_REQUIRE(out_dtype == MOE_DTYPE_F32 || out_dtype == MOE_DTYPE_F16 ||
                  out_dtype == MOE_DTYPE_BF16,
              MOE_ERR_INVALID_ARG, "fp8_matmul: out dtype must be f32/f16/bf16");
  KSW_REQUIRE(ld_x >= inner && ld_w >= inner && ld_out >= out_cols &&
                  (addend == nullptr || ld_addend >= out_cols),
              MOE_ERR_INVALID_ARG, "fp8_matmul: row stride shorter than a row");
  KSW_REQUIRE(ld_x % 16 == 0 && ld_w % 16 == 0 && aligned16(x) && aligned16(w),
              MOE_ERR_INVALID_ARG,
              "fp8_matmul: the fp8 rows must start on 16-byte boundaries");
  int sms = 0;
  if ((st = check_device(&sms)) != MOE_OK) return st;
  if (num_rows == 0) return MOE_OK;
  KSW_REQUIRE(x && x_scale && w && w_scale && out, MOE_ERR_INVALID_ARG,
              "fp8_matmul: null pointer");
  const bool mx = scale_format == 1;
  const Plan plan = plan_matmul(num_rows, out_cols, inner, mx, sms);
  CUtensorMap tx, tw;
  const uint32_t x_box = plan.rows ? kLanes : uint32_t(plan.bn);
  const uint32_t w_box = plan.rows ? uint32_t(plan.bn) : kLanes;
  st = encode_tma_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, uint64_t(inner),
                     uint64_t(num_rows), uint64_t(ld_x), kKB, x_box);
  if (st != MOE_OK) return st;
  st = encode_tma_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, uint64_t(inner),
                     uint64_t(out_cols), uint64_t(ld_w), kKB, w_box);
  if (st != MOE_OK) return st;
  MatmulParams p = {};
  p.xs = x_scale;
  p.xs_row = xs_row_stride;
  p.xs_blk = xs_block_stride;
  p.ws = w_scale;
  p.out = out;
  p.ld_out = ld_out;
  p.add = addend;
  p.ld_add = addend ? ld_addend : 0;
  p.T = num_rows;
  p.N = out_cols;
  p.kb_total = int(ceil_div(inner, kKB));
  p.t_tiles = int(ceil_div(num_rows, plan.rows ? kLanes : plan.bn));
  p.n_tiles = int(ceil_div(out_cols, plan.rows ? plan.bn : kLanes));
  p.splits = plan.splits;
  p.status = status;
  p.wait_limit_ns = kWaitLimitNs;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (out_dtype == MOE_DTYPE_F32) return run_matmul<float>(plan, mx, tw, tx, p, s);
  if (out_dtype == MOE_DTYPE_BF16) return run_matmul<__nv_bfloat16>(plan, mx, tw, tx, p, s);
  return run_matmul<__half>(plan, mx, tw, tx, p, s);
}
