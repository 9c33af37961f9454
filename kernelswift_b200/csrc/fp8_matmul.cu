// Dense block-scaled fp8 product
//   out[t, n] = addend[t, n] + sum_kb sx[t, kb] sw[n / 128, kb]
//                              sum_{k in block kb} xq[t, k] wq[n, k]
// with e4m3 operands xq [T, K] and wq [N, K] on the tcgen05 tensor cores.
//
// UE8M0 scales are applied by the tensor core (kind::mxf8f6f4, block_scale):
// all k-blocks of a tile accumulate in one TMEM accumulator. fp32 scales
// cannot be: each k-block's product goes to a TMEM buffer of its own and is
// added to fp32 registers times sx * sw. Two kernels:
//
// fp8_cols_kernel: a tile is 128 weight rows (TMEM lanes) x BN tokens
//   (columns), BN in {16, ..., 256}, so that a handful of tokens costs a
//   handful of columns. For fp32 scales a warp brings sx * sw of every column
//   to shared memory per k-block (a column's factor is the same for all
//   lanes). Tiles too few for the SMs are split along K over a cluster of up
//   to 8 CTAs, whose fp32 partials are summed in rank order through
//   distributed shared memory: one launch, no workspace, a fixed order.
//   Bound by the stream of weights and, at a few MB of them, by the fixed cost
//   of a launch (about 3 us of barrier, TMEM and cluster set-up, pipeline fill
//   and the last tile's way out). One B200, back to back, UE8M0: 1 x 4096 x 7168
//   8.8 us (3.3 TB/s), 1 x 36864 x 7168 40.6 us (6.5 TB/s), 16 x 7168 x 2048 6.6
//   us, 128 x 4096 x 7168 13.6 us; fp32 scales 8.9, 42, 6.9 and 15.3 us.
//
// fp8_pair_kernel: many tokens. Two CTAs share a tile of 256 tokens (lanes) x
//   256 weight rows (columns), each holding half of either operand; with fp32
//   scales a thread's columns share one sw and its row one sx, a single factor
//   per thread and k-block. Bound by the tensor core at the clock that the power
//   limit leaves (UE8M0), or by the way of a k-block's product through tensor
//   memory and registers (fp32 scales). One B200, back to back, UE8M0: 4096 x
//   4096 x 7168 88 us (2740 TFLOP/s), 16384 x 4096 x 7168 369 to 393 us (by the
//   clock), 8192 x 7168 x 2048 94 us; fp32 scales 122 us (1980 TFLOP/s), 505 us and
//   139 us. Tiles of 256 x 256 take an SM's shared memory 512 cycles per k-block for
//   the 512 of its MMAs; 128 x 256 tiles of single CTAs would take 768.
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "runtime.h"

namespace ksw {
namespace {

constexpr int kKB = 128;            // bytes (= columns) of a k-block
constexpr int kLanes = 128;         // rows of the MMA
constexpr int kABytes = kLanes * kKB;
constexpr int kFacSlots = 8;        // fp32 scale ring: k-blocks

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
  int slice;               // tokens that each of them sums (kPush): a multiple of 4
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
// Shared-memory address `addr` of this CTA in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
// Stores 16 bytes into a CTA of the cluster; they are counted on its barrier.
__device__ __forceinline__ void st_async4(uint32_t addr, const float* v, uint32_t bar) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, "
      "[%5];" ::"r"(addr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
      "r"(__float_as_uint(v[3])), "r"(bar)
      : "memory");
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

// One lane of the (converged) warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(0xffffffffu, ok); }
// Barrier `id` of 128 threads; whether all of them came with `ok`. A warp that
// gave up waiting takes part with false, so none is left at the barrier alone.
__device__ __forceinline__ bool group_ok(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
      "bar.red.and.pred p, %1, 128, q;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(uint32_t(ok))
      : "memory");
  return r != 0;
}

// Waits for this thread's tensor-memory loads; the values read pass through
// the (empty) statements after it, so no use of them can move before it.
template <int N>
__device__ __forceinline__ void tmem_arrived(uint32_t (&v)[N]) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}

// The slots of a ring that have been filled, and the parity of each one's last
// fill (whichever warp's), so that a block ends only after what it caused: the
// copies into a stage (drain), and the MMAs' last arrivals on the ring's `empty`
// barriers (released). tcgen05.commit arrives asynchronously, for a CTA pair on
// the other CTA's barriers too; the MMAs' completion alone (final_bar) does not say
// that earlier arrivals have landed, and one that came late would land in the
// shared memory of the SM's next block. A slot's k-th fill and its k-th release
// complete phases of one parity. When a wait gave up, `released` does not wait.
struct Filled {
  uint32_t used = 0, parity = 0;
  __device__ __forceinline__ void add(int stage, uint32_t phase) {
    used |= 1u << stage;
    parity = (parity & ~(1u << stage)) | (phase << stage);
  }
  __device__ __forceinline__ void drain(uint64_t* full, int stages, uint64_t limit) const {
    volatile int no_abort = 0;
    released(full, stages, &no_abort, limit);
  }
  __device__ __forceinline__ void released(uint64_t* bars, int slots, volatile int* abort,
                                           uint64_t limit) const {
    for (int s = 0; s < slots; ++s)
      if ((used >> s) & 1u) mbar_wait_bounded(&bars[s], (parity >> s) & 1u, abort, limit);
  }
};

// Asks L2 to fetch the box at (c0, c1); nothing reaches the SM, nothing waits.
__device__ __forceinline__ void l2_prefetch_2d(const CUtensorMap* tm, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(tm)),
               "r"(c0), "r"(c1)
               : "memory");
}
// k-blocks of weights that a CTA asks L2 for while its predecessor still runs, UE8M0
// and fp32 scales: 1 x 4096 x 7168 9.5 and 9.8 us without, 8.8 and 8.9 with 6 (about
// what fits in the ring), 8.9 and 9.1 with 16; 16 x 7168 x 2048 6.9 and 7.2, 6.6 and
// 6.9, 6.6 and 6.9. Of many columns a ring holds fewer k-blocks: 128 x 4096 x 7168
// 13.2 and 15.5, 13.6 and 15.3, 14.7 and 16.5.
constexpr int kL2Ahead = 6;

// Asks L2 for the line at `p`.
__device__ __forceinline__ void l2_prefetch(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory");
}

// TMA producers: two warps take the stages in turn. A turn (wait for the
// stage, announce its bytes, issue two copies) takes a warp about 490 cycles
// whatever the boxes' size (570 from a single diverged lane), and a stage's
// MMAs no more than 512, so one warp alone would starve the tensor core.
constexpr int kProducers = 2;
__device__ __forceinline__ int producer_of(int warp) { return warp == 0 ? 0 : warp == 3 ? 1 : -1; }

// UE8M0 scales travel as words of four bytes, the scales of one row in a quad
// of k-blocks. A loader warp builds the tensor core's 512-byte chunks (128
// rows: lane l holds rows l, l + 32, l + 64, l + 96) of Q quads at a time.
template <int Q>
struct ScaleWords {
  uint32_t v[4][Q];

  // The words of quads q0 .. q0 + Q of the 128 rows of `scale` from row0 on.
  // Rows at or past `rows` and quads past the last repeat the last one (their
  // products are never stored, or never made), so that all loads are
  // unconditional and under way together: loaded one by one behind branches
  // they took 2,000 to 3,600 cycles a quad, and a quad's MMAs take 2,048.
  __device__ __forceinline__ void fetch(const uint8_t* scale, int64_t row_stride,
                                        int64_t blk_stride, bool words, int64_t row0,
                                        int64_t rows, int lane, int q0, int kb) {
    const uint8_t* at[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      at[r] = scale + min(row0 + 32 * r + lane, rows - 1) * row_stride;
    if (words) {
      const int last = kb / 4 - 1;  // whole words
#pragma unroll
      for (int j = 0; j < Q; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r][j] = __ldg(reinterpret_cast<const uint32_t*>(at[r]) + min(q0 + j, last));
    }
    // quads with fewer than four blocks, and scales that are not in words
#pragma unroll
    for (int j = 0; j < Q; ++j) {
      const int b = 4 * (q0 + j);
      if (b < kb && (!words || b + 4 > kb)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint32_t w = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w |= uint32_t(__ldg(at[r] + min(b + i, kb - 1) * blk_stride)) << (8 * i);
          v[r][j] = w;
        }
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* chunk, int stride, int lane) const {
#pragma unroll
    for (int j = 0; j < Q; ++j)
      reinterpret_cast<uint4*>(chunk + j * stride)[lane] =
          make_uint4(v[0][j], v[1][j], v[2][j], v[3][j]);
  }
};

// The same of one 128-row block of the weights, whose rows share their scale:
// lane i < 4 Q holds byte i.
template <int Q>
struct BlockWords {
  uint32_t byte;
  __device__ __forceinline__ void fetch(const uint8_t* block, bool in, int lane, int q0, int kb) {
    const int b = 4 * q0 + lane;
    byte = in && lane < 4 * Q && b < kb ? __ldg(block + b) : 0u;
  }
  __device__ __forceinline__ void store(uint8_t* chunk, int stride, int lane) const {
#pragma unroll
    for (int j = 0; j < Q; ++j) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= __shfl_sync(0xffffffffu, byte, 4 * j + i) << (8 * i);
      reinterpret_cast<uint4*>(chunk + j * stride)[lane] = make_uint4(w, w, w, w);
    }
  }
};

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
  // UE8M0 scale ring: slots, and quads of k-blocks in each. A short run of
  // k-blocks (a split tile's) starts sooner on small slots.
  static constexpr int kSfSlots = 4, kQuads = 1;
  static constexpr int kQuadBytes = 512 * (1 + kSfb);
  static constexpr int kRingBytes =
      MX ? kSfSlots * kQuads * kQuadBytes : kFacSlots * BN * 4;
  static constexpr int kGroups = kEpiWarps / 4;       // epilogue groups of 128 lanes
  // A split tile's partials: pushed into the memory of the CTA that sums them
  // where that costs no pipeline stages (BN <= 32), else read from their own
  // CTA's memory between two cluster barriers (UE8M0, 16 x 4096 x 7168 9.5 us read,
  // 9.3 pushed; 16 x 7168 x 2048 6.9 and 6.6; 1 x 4096 x 7168 8.95 and 8.75).
  static constexpr bool kPush = BN <= 32;
  static constexpr int kRecvBytes = kPush ? 16384 : 0;
  static constexpr int kOutBytes =  // staged output, or received partials
      kGroups * 2 * kStagedBytes > kRecvBytes ? kGroups * 2 * kStagedBytes : kRecvBytes;
  static constexpr size_t kFixed = 1024 + 512 + kRingBytes + size_t(kOutBytes);
  static constexpr int kStages = int(((kCtas == 2 ? 112 : 224) * 1024 - kFixed) / kStageBytes);
  static constexpr size_t kSmem = kFixed + size_t(kStages) * kStageBytes;
  // TMEM: accumulators (UE8M0) or per-k-block buffers (fp32), then scale slots
  static constexpr int kBufs = MX ? (BN == 256 ? 1 : 2) : 4;
  static constexpr int kSfCol0 = kBufs * BN;
  static constexpr int kSfCols = 4 * (1 + kSfb);
  static constexpr int kUsed = kSfCol0 + (MX ? kSfSlots * kQuads * kSfCols : 0);
  static constexpr int kTmem = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(kUsed <= 512 && kTmem * kCtas <= 512, "TMEM columns");
  static_assert(size_t(kStages) * kStageBytes >= size_t(BN) * kLanes * 4,
                "the partial tile reuses the stages");
  static_assert(8 * (2 * kStages + 2 * kFacSlots + 2 * 4 + 2) + 8 <= 512, "barriers");
};

template <bool MX, int BN, typename TOUT>
__global__ void __launch_bounds__(ColsCfg<MX, BN>::kThreads, ColsCfg<MX, BN>::kCtas)
    fp8_cols_kernel(const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmX, const MatmulParams p) {
  using C = ColsCfg<MX, BN>;
  constexpr int STAGES = C::kStages;
  constexpr int NB = C::kBufs;
  constexpr int COLS = C::kCols;
  constexpr int SLOTS = MX ? C::kSfSlots : kFacSlots;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * kABytes;
  uint8_t* sRing = sB + STAGES * C::kBBytes;
  uint8_t* sOut = sRing + C::kRingBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + C::kOutBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* sfull = empty + STAGES;
  uint64_t* sempty = sfull + SLOTS;
  uint64_t* tfull = sempty + SLOTS;
  uint64_t* tempty = tfull + NB;
  uint64_t* final_bar = tempty + NB;
  uint64_t* recv_bar = final_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(recv_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  // the warp's number, known to be the same for all its lanes
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const bool push = C::kPush && p.splits > 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&sfull[s], 1);
      mbar_init(&sempty[s], MX ? 1 : C::kEpiWarps);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], C::kEpiWarps);
    }
    mbar_init(final_bar, 1);
    mbar_init(recv_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmW);  // kernel arguments, no predecessor's data
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (push) {
    __syncwarp();
    cluster_sync();  // every CTA's recv_bar is ready
  }

  const uint64_t limit = p.wait_limit_ns;
  const int tiles = p.t_tiles * p.n_tiles;
  // a cluster's CTAs share a tile: CTA `part` takes k-blocks [kb0, kb1)
  const int part = int(blockIdx.x) % p.splits;
  const int first = int(blockIdx.x) / p.splits, step = int(gridDim.x) / p.splits;
  const int kb0 = int(int64_t(p.kb_total) * part / p.splits);
  const int kb1 = int(int64_t(p.kb_total) * (part + 1) / p.splits);
  // While the previous kernel finishes, the weights of this CTA's first tile
  // start on their way to L2. Should that kernel be writing them, no harm is
  // done: nothing is read before the wait, and L2 is where its writes land.
  if (warp == 0 && first < tiles && elect_one()) {
    const int row = tile_at(first, p.t_tiles, p.n_tiles).n * kLanes;
    for (int kb = kb0; kb < min(kb1, kb0 + kL2Ahead); ++kb) l2_prefetch_2d(&tmW, kb * kKB, row);
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();

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
      // past the last token or column the last one again, so that the loads are
      // unconditional and go out together
      const TOUT* add = static_cast<const TOUT*>(p.add) + min(t0, p.T - 1) * p.ld_add +
                        min(n0 + row, p.N - 1);
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        TOUT a[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          a[j] = *add;
          add += c + j + 1 < live ? p.ld_add : 0;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[c + j] += to_f32(a[j]);
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
    // the next tile starts with buffer 0 again, after its own group_ok
  };

  if (producer_of(warp) >= 0) {
    // ---------------- TMA producers ----------------
    const bool leader = elect_one();
    const int mine = producer_of(warp);
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    Filled filled;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (turn == mine) {
          ok = all_ok(mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag, limit));
          if (!ok) break;
          if (leader) {
            mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
            tma_load_2d(sA + stage * kABytes, &tmW, kb * kKB, tile.n * kLanes, &full[stage]);
            tma_load_2d(sB + stage * C::kBBytes, &tmX, kb * kKB, tile.t * BN, &full[stage]);
          }
          __syncwarp();
        }
        filled.add(stage, phase);
        turn = turn + 1 == kProducers ? 0 : turn + 1;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    filled.drain(full, STAGES, limit);
    filled.released(empty, STAGES, abort_flag, limit);
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // The whole warp walks the loop and one lane issues: operands computed by
    // a converged warp stay in uniform registers, where the MMA takes them.
    const bool leader = elect_one();
    const uint64_t desc_a = make_sw128_desc(smem_u32(sA));
    const uint64_t desc_b = make_sw128_desc(smem_u32(sB));
    int stage = 0, buf = 0, slot = 0;
    [[maybe_unused]] uint32_t sf = 0;  // TMEM of the quad's scales
    uint32_t phase = 0, bphase = 0, sphase = 0;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      if constexpr (MX) {
        if (!all_ok(mbar_wait_bounded(&tempty[buf], bphase ^ 1u, abort_flag, limit))) break;
        tc_fence_after();
      }
      for (int kb = kb0; kb < kb1; ++kb) {
        if constexpr (MX) {
          if (kb == kb0 || kb % (4 * C::kQuads) == 0) {
            ok = all_ok(mbar_wait_bounded(&sfull[slot], sphase, abort_flag, limit));
            if (!ok) break;
            tc_fence_after();
          }
          if (kb == kb0 || (kb & 3) == 0) {
            // a slot's TMEM columns are rewritten only after sempty, i.e. after
            // the MMAs that read them completed
            const int quad = slot * C::kQuads + (kb >> 2) % C::kQuads;
            sf = tmem_base + uint32_t(C::kSfCol0 + quad * C::kSfCols);
            const uint32_t src = smem_u32(sRing + quad * C::kQuadBytes);
            if (leader) {
#pragma unroll
              for (int c = 0; c < 1 + C::kSfb; ++c)
                tc_cp_sf(sf + 4 * c, make_sf_desc(src + 512 * c));
            }
            __syncwarp();
          }
        } else {
          ok = all_ok(mbar_wait_bounded(&tempty[buf], bphase ^ 1u, abort_flag, limit));
          if (!ok) break;
        }
        ok = all_ok(mbar_wait_bounded(&full[stage], phase, abort_flag, limit));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem_base + uint32_t(buf * BN);
        // descriptors of the stage's tiles; 32 bytes further along K are 2 units
        const uint64_t a0 = desc_a + uint32_t(stage * (kABytes / 16));
        const uint64_t b0 = desc_b + uint32_t(stage * (C::kBBytes / 16));
        if constexpr (MX) {
          const uint32_t idesc = idesc_sf_ids(make_idesc_mx(kLanes, BN), uint32_t(kb & 3));
          const bool slot_end = kb + 1 == kb1 || (kb + 1) % (4 * C::kQuads) == 0;
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_mx(d, a0 + 2 * kk, b0 + 2 * kk, idesc, sf, sf + 4,
                        (kb > kb0 || kk > 0) ? 1u : 0u);
            tc_commit(&empty[stage]);
            if (slot_end) tc_commit(&sempty[slot]);
          }
          __syncwarp();
          if (slot_end) {
            if (++slot == SLOTS) {
              slot = 0;
              sphase ^= 1u;
            }
          }
        } else {
          constexpr uint32_t idesc = make_idesc(1u, 0u, kLanes, BN);
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma<kKindF8>(d, a0 + 2 * kk, b0 + 2 * kk, idesc, kk > 0 ? 1u : 0u);
            tc_commit(&empty[stage]);
            tc_commit(&tfull[buf]);
          }
          __syncwarp();
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
        if (leader) tc_commit(&tfull[buf]);
        __syncwarp();
        if (++buf == NB) {
          buf = 0;
          bphase ^= 1u;
        }
      }
    }
    if (leader) tc_commit(final_bar);
    volatile int no_abort = 0;
    mbar_wait_bounded(final_bar, 0, &no_abort, limit);
  } else if (warp == 2) {
    // ---------------- scales ----------------
    int slot = 0;
    uint32_t sphase = 0;
    bool ok = true;
    if constexpr (MX) {
      constexpr int Q = C::kQuads;
      const uint8_t* xs = static_cast<const uint8_t*>(p.xs);
      const bool words = p.kb_total >= 4 && p.xs_blk == 1 && p.xs_row % 4 == 0 &&
                         (reinterpret_cast<uintptr_t>(xs) & 3) == 0;
      const int q_first = kb0 / 4 / Q * Q, q_end = (kb1 + 3) / 4;
      ScaleWords<Q> xw[C::kSfb];
      BlockWords<Q> ww;
      auto fetch = [&](int i, int q0) {
        const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
#pragma unroll
        for (int c = 0; c < C::kSfb; ++c) {
          const int64_t t0 = int64_t(tile.t) * BN + 128 * c;
          xw[c].fetch(xs, p.xs_row, p.xs_blk, words, t0, min(p.T, t0 + BN), lane, q0, p.kb_total);
        }
        ww.fetch(static_cast<const uint8_t*>(p.ws) + int64_t(tile.n) * p.kb_total, true, lane, q0,
                 p.kb_total);
      };
      Filled filled;
      if (first < tiles) fetch(first, q_first);
      for (int i = first; ok && i < tiles; i += step) {
        for (int q0 = q_first; q0 < q_end; q0 += Q) {
          ok = all_ok(mbar_wait_bounded(&sempty[slot], sphase ^ 1u, abort_flag, limit));
          if (!ok) break;
          uint8_t* dst = sRing + slot * Q * C::kQuadBytes;
          ww.store(dst, C::kQuadBytes, lane);
#pragma unroll
          for (int c = 0; c < C::kSfb; ++c) xw[c].store(dst + 512 * (1 + c), C::kQuadBytes, lane);
          // the copies to tensor memory read it through the async proxy
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull[slot]);
          filled.add(slot, sphase);
          // the next words' loads run while the slots ahead are used
          if (q0 + Q < q_end)
            fetch(i, q0 + Q);
          else if (i + step < tiles)
            fetch(i + step, q_first);
          if (++slot == SLOTS) {
            slot = 0;
            sphase ^= 1u;
          }
        }
      }
      filled.released(sempty, SLOTS, abort_flag, limit);
    } else {
      // sx * sw of four k-blocks at a time, loaded together and a turn ahead
      constexpr int R = (BN + 31) / 32, U = 4;
      const float* xs = static_cast<const float*>(p.xs);
      float v[U][R];
      auto fetch = [&](int i, int k0) {
        const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
        const float* ws = static_cast<const float*>(p.ws) + int64_t(tile.n) * p.kb_total;
        const float* at[R];
#pragma unroll
        for (int r = 0; r < R; ++r)  // tokens past the last one repeat it
          at[r] = xs + min(int64_t(tile.t) * BN + 32 * r + lane, p.T - 1) * p.xs_row;
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int kb = min(k0 + u, kb1 - 1);
          w[u] = __ldg(ws + kb);
#pragma unroll
          for (int r = 0; r < R; ++r) v[u][r] = __ldg(at[r] + kb * p.xs_blk);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) v[u][r] *= w[u];
      };
      if (first < tiles) fetch(first, kb0);
      for (int i = first; ok && i < tiles; i += step) {
        for (int k0 = kb0; ok && k0 < kb1; k0 += U) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (k0 + u >= kb1) break;
            ok = all_ok(mbar_wait_bounded(&sempty[slot], sphase ^ 1u, abort_flag, limit));
            if (!ok) break;
            float* dst = reinterpret_cast<float*>(sRing) + slot * BN;
#pragma unroll
            for (int r = 0; r < R; ++r)
              if (32 * r + lane < BN) dst[32 * r + lane] = v[u][r];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sfull[slot]);
            if (++slot == SLOTS) {
              slot = 0;
              sphase ^= 1u;
            }
          }
          if (k0 + U < kb1)
            fetch(i, k0 + U);
          else if (i + step < tiles)
            fetch(i + step, kb0);
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------- promotion and epilogue ----------------
    const int row = (warp & 3) * 32 + lane;
    const int group = (warp - 4) >> 2;
    const int col0 = group * COLS;
    const uint32_t lane_base = tmem_base + (uint32_t((warp & 3) * 32) << 16) + uint32_t(col0);
    int buf = 0, slot = 0;
    uint32_t bphase = 0, sphase = 0;
    constexpr int BATCH = COLS >= 32 ? 32 : 16;
    if (push && threadIdx.x == 128) {
      const int64_t t0 = int64_t(tile_at(first, p.t_tiles, p.n_tiles).t) * BN + part * p.slice;
      if (part * p.slice < BN && t0 < p.T)
        mbar_arrive_expect_tx(recv_bar, uint32_t(p.splits * p.slice * kLanes * 4));
    }
    for (int i = first; epi_ok && i < tiles; i += step) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      if (p.add != nullptr) {
        // the tile's addend is in L2 by the time its sums are done: a lane asks for
        // the warp's 32 columns of a token
        const int64_t n = int64_t(tile.n) * kLanes + (warp & 3) * 32;
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          const int64_t t = int64_t(tile.t) * BN + col0 + c + lane;
          if (c + lane < COLS && t < p.T && n < p.N)
            l2_prefetch(static_cast<const TOUT*>(p.add) + t * p.ld_add + n);
        }
      }
      if constexpr (MX) {
        epi_ok = group_ok(1 + group, mbar_wait_bounded(&tfull[buf], bphase, abort_flag, limit));
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
        epi_ok = group_ok(1 + group, epi_ok);
        if (!epi_ok) break;
      }
      if (p.splits == 1) {
        store_tile(tile, col0, row, group);
      } else if constexpr (C::kPush) {
        // tokens [o * ts, (o + 1) * ts) go to CTA o of the cluster, as
        // [source][weight row][token]
        const int ts = p.slice;
        const int live = int(min(int64_t(BN), p.T - int64_t(tile.t) * BN));
        const uint32_t dst = smem_u32(sOut) + 4u * uint32_t((part * kLanes + row) * ts);
        const uint32_t bar = smem_u32(recv_bar);
#pragma unroll
        for (int j = 0; j < COLS; j += 4) {
          const int o = j / ts;
          if (o * ts < live)
            st_async4(peer_addr(dst + 4u * uint32_t(j - o * ts), uint32_t(o)), &acc[j],
                      peer_addr(bar, uint32_t(o)));
        }
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
  if (push) {
    // a CTA leaves once all have arrived here, their stores to it on the way
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const Tile tile = tile_at(first, p.t_tiles, p.n_tiles);
    const int64_t n = int64_t(tile.n) * kLanes + (threadIdx.x & 127);
    const int ts = p.slice, j0 = part * ts;
    const int64_t t0 = int64_t(tile.t) * BN + j0;
    if (warp >= 4 && j0 < BN && t0 < p.T) {
      // four tokens of the addend at a time, ahead of the sums they go to
      const TOUT* add = static_cast<const TOUT*>(p.add) + min(n, p.N - 1);
      TOUT a[4];
      auto fetch = [&](int j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = add[min(t0 + j + e, p.T - 1) * p.ld_add];
      };
      if (p.add != nullptr) fetch(0);
      bool ok = mbar_wait_bounded(recv_bar, 0, abort_flag, limit);
      if (all_ok(ok) && !*abort_flag && n < p.N) {
        const float4* src = reinterpret_cast<const float4*>(sOut) + (threadIdx.x & 127) * (ts / 4);
        for (int j = 0; j < ts; j += 4) {
          float4 sum = src[j / 4];
          for (int r = 1; r < p.splits; ++r) {  // in rank order
            const float4 v = src[r * kLanes * (ts / 4) + j / 4];
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
          }
          float out[4] = {sum.x, sum.y, sum.z, sum.w};
          if (p.add != nullptr) {
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] += to_f32(a[e]);
            if (j + 4 < ts) fetch(j + 4);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t t = t0 + j + e;
            if (j0 + j + e < BN && t < p.T)
              static_cast<TOUT*>(p.out)[t * p.ld_out + n] = from_f32<TOUT>(out[e]);
          }
        }
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __syncthreads();
  if (p.splits > 1 && !push) {
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
        float a = 0.0f;
        if (p.add != nullptr)
          a = to_f32(static_cast<const TOUT*>(p.add)[t * p.ld_add + min(n, p.N - 1)]);
        float v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          v[r] = r < p.splits ? ld_peer(base + uint32_t(j * kLanes * 4), uint32_t(r)) : 0.0f;
        float sum = v[0];
#pragma unroll
        for (int r = 1; r < 8; ++r) sum += v[r];
        if (p.add != nullptr) sum += a;
        if (n < p.N) static_cast<TOUT*>(p.out)[t * p.ld_out + n] = from_f32<TOUT>(sum);
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
// fp8_pair_kernel: a pair of CTAs (cta_group::2) per tile of 256 tokens x 256
// weight rows. CTA r of the pair holds tokens 128 r .. (its TMEM lanes) and
// loads weight rows 128 r .. of the tile; the even CTA issues the MMAs, which
// read both halves of the weights for both CTAs. Per k-block a CTA takes in
// and feeds 32 KB instead of the 48 KB of a 128 x 256 tile of its own, which
// needs 768 cycles of shared-memory bandwidth for the MMA's 512.
// ---------------------------------------------------------------------------
template <bool MX, bool VEC>
struct PairCfg {
  static constexpr int kBN = 256;
  static constexpr int kEpiWarps = MX ? 16 : 8;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kCols = kBN / (kEpiWarps / 4);  // per epilogue warp: 64 or 128
  // fp32 scales: a k-block's product is two MMAs of 128 columns, each with its
  // own issuing warp, buffers and barriers, so that four buffers of 128 columns
  // hide the way from an MMA's end to its buffer's release
  static constexpr int kHalves = MX ? 1 : 2;
  static constexpr int kN = kBN / kHalves;             // columns of an MMA
  static constexpr int kBox = kN / 2;                  // weight rows of a CTA's TMA box
  static constexpr int kBBytes = kBN / 2 * kKB;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = MX && !VEC ? 5 : 6;
  static constexpr int kSfbChunks = kBN / 128;
  static constexpr int kSfSlots = 2, kQuads = 4;  // scale ring: slots, quads in each
  static constexpr int kQuadBytes = 512 * (1 + kSfbChunks);
  static constexpr int kRingBytes = MX ? kSfSlots * kQuads * kQuadBytes : 0;
  // VEC: rows of the output (and the addend) in whole 16-byte vectors. Without
  // it a warp passes 32 rows x 64 bytes at a time through a piece of shared
  // memory, rows 17 words apart.
  static constexpr int kRunBytes = 64, kPitchBytes = kRunBytes + 4;
  static constexpr int kStageOut = VEC ? 0 : 32 * kPitchBytes;
  static constexpr size_t kSmem =
      1024 + 512 + kRingBytes + kEpiWarps * kStageOut + size_t(kStages) * kStageBytes;
  static_assert(kSmem <= 232448, "shared memory of an SM");
  // TMEM: one accumulator and the scale slots (UE8M0), or two k-block buffers
  static constexpr int kBufs = MX ? 1 : 2;
  static constexpr int kSfCol0 = kBufs * kBN;
  static constexpr int kSfCols = 4 * (1 + kSfbChunks);
  static_assert(kSfCol0 + (MX ? kSfSlots * kQuads * kSfCols : 0) <= 512, "TMEM columns");
  static_assert(8 * (2 * kStages + 2 * kSfSlots + 2 * kBufs * kHalves + 1) + 8 <= 512,
                "barriers");
  // fp32 scales: the block launches at kLaunchRegs registers per thread; the
  // control warpgroup gives registers back and the 8 epilogue warps take them,
  // for 128 sums and a batch of 64 partials each. The split adds up to the
  // launch's total, which the host checks against the compiled kernel.
  static constexpr int kLaunchRegs = 168, kCtrlRegs = 72, kEpiRegs = 216;
  static_assert(MX || 128 * kCtrlRegs + 32 * kEpiWarps * kEpiRegs == kThreads * kLaunchRegs,
                "setmaxnreg split");
};

// Arrives on a barrier of the cluster, after this thread's (and, after a warp
// barrier, its warp's) writes.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
               : "memory");
}
// The same where no memory is handed over but tensor memory that has been
// read: the cluster-wide release would wait for unrelated loads and stores.
__device__ __forceinline__ void mbar_arrive_cluster_read(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// mbar_wait_bounded for a phase that threads of the other CTA complete too.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "n"(kMbarSuspendHintNs)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity,
                                                  volatile int* abort, uint64_t limit_ns) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if (*abort) return false;
    if (globaltimer_ns() - t0 > limit_ns) {
      *abort = 1;
      return false;
    }
  }
}
// TMA load into this CTA whose bytes are counted on the even CTA's barrier.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* tm, int32_t c0,
                                              int32_t c1, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(leader_bar)
      : "memory");
}
// Arrives on `bar` of both CTAs when the MMAs issued so far have completed.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"(uint16_t(3))
      : "memory");
}
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_mx_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                               uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
      : "memory");
}
// Scale chunk at the same shared-memory offset of each CTA into its own TMEM.
__device__ __forceinline__ void tc_cp_sf_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc)
               : "memory");
}

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

template <bool MX, bool VEC, typename TOUT>
__global__ void __launch_bounds__(PairCfg<MX, VEC>::kThreads, 1)
    fp8_pair_kernel(const __grid_constant__ CUtensorMap tmX,
                    const __grid_constant__ CUtensorMap tmW, const MatmulParams p) {
  using C = PairCfg<MX, VEC>;
  constexpr int STAGES = C::kStages;
  constexpr int NB = C::kBufs;
  constexpr int COLS = C::kCols;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * kABytes;
  uint8_t* sRing = sB + STAGES * C::kBBytes;
  uint8_t* sOut = sRing + C::kRingBytes;
  uint64_t* full =
      reinterpret_cast<uint64_t*>(sOut + C::kEpiWarps * C::kStageOut);  // used in the even CTA
  uint64_t* empty = full + STAGES;
  uint64_t* sfull = empty + STAGES;  // used in the even CTA
  uint64_t* sempty = sfull + C::kSfSlots;
  uint64_t* tfull = sempty + C::kSfSlots;
  uint64_t* tempty = tfull + NB * C::kHalves;  // used in the even CTA
  uint64_t* final_bar = tempty + NB * C::kHalves;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(final_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  // the warp's number, known to be the same for all its lanes
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1;  // in the pair
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], C::kHalves);
    }
    for (int s = 0; s < C::kSfSlots; ++s) {
      mbar_init(&sfull[s], 2);
      mbar_init(&sempty[s], 1);
    }
    for (int b = 0; b < NB * C::kHalves; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * C::kEpiWarps / C::kHalves);
    }
    mbar_init(final_bar, C::kHalves);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // both CTAs' barriers and TMEM are ready
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();
  const uint64_t limit = p.wait_limit_ns;
  const int tiles = p.t_tiles * p.n_tiles;
  const int kbs = p.kb_total;
  const int first = int(blockIdx.x) >> 1, step = int(gridDim.x) >> 1;

  if (!MX && warp < 4) setmaxnreg_dec<C::kCtrlRegs>();
  if (producer_of(warp) >= 0) {
    // ---------------- TMA producers of this CTA's halves ----------------
    const bool leader = elect_one();
    if (leader) {
      tma_prefetch_desc(&tmX);
      tma_prefetch_desc(&tmW);
    }
    const int mine = producer_of(warp);
    const uint32_t bars = peer_addr(smem_u32(full), 0);  // the even CTA's
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    Filled filled;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      const int x_row = tile.t * 256 + int(rank) * kLanes;
      const int w_row = tile.n * C::kBN + int(rank) * C::kBox;
      for (int kb = 0; kb < kbs; ++kb) {
        if (turn == mine) {
          ok = all_ok(mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag, limit));
          if (!ok) break;
          if (leader) {
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::kStageBytes);
            const uint32_t bar = bars + 8u * uint32_t(stage);
            tma_load_pair(sA + stage * kABytes, &tmX, kb * kKB, x_row, bar);
#pragma unroll
            for (int h = 0; h < C::kHalves; ++h)
              tma_load_pair(sB + stage * C::kBBytes + h * C::kBox * kKB, &tmW, kb * kKB,
                            w_row + h * C::kN, bar);
          }
          __syncwarp();
        }
        filled.add(stage, phase);
        turn = turn + 1 == kProducers ? 0 : turn + 1;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // the even CTA's barriers count both CTAs' bytes; the odd CTA stays until
    // the cluster barrier below
    if (rank == 0) filled.drain(full, STAGES, limit);
    filled.released(empty, STAGES, abort_flag, limit);
  } else if (warp >= 1 && warp <= C::kHalves && rank == 0) {
    // ---------------- MMA issuers, for both CTAs ----------------
    // The whole warp walks the loop and one lane issues: operands computed by
    // a converged warp stay in uniform registers, where the MMA takes them.
    const bool leader = elect_one();
    const int half = warp - 1;
    const uint64_t desc_a = make_sw128_desc(smem_u32(sA));
    const uint64_t desc_b = make_sw128_desc(smem_u32(sB + half * C::kBox * kKB));
    uint64_t* const my_tfull = tfull + half * NB;
    uint64_t* const my_tempty = tempty + half * NB;
    int stage = 0, buf = 0, slot = 0;
    [[maybe_unused]] uint32_t sf = 0;  // TMEM of the quad's scales
    uint32_t phase = 0, bphase = 0, sphase = 0;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      if constexpr (MX) {
        if (!all_ok(mbar_wait_bounded(&my_tempty[buf], bphase ^ 1u, abort_flag, limit))) break;
        tc_fence_after();
      }
      for (int kb = 0; kb < kbs; ++kb) {
        if constexpr (MX) {
          if (kb % (4 * C::kQuads) == 0) {
            ok = all_ok(mbar_wait_cluster(&sfull[slot], sphase, abort_flag, limit));
            if (!ok) break;
            tc_fence_after();
          }
          if ((kb & 3) == 0) {
            const int quad = slot * C::kQuads + (kb >> 2) % C::kQuads;
            sf = tmem_base + uint32_t(C::kSfCol0 + quad * C::kSfCols);
            const uint32_t src = smem_u32(sRing + quad * C::kQuadBytes);
            if (leader) {
#pragma unroll
              for (int c = 0; c < 1 + C::kSfbChunks; ++c)
                tc_cp_sf_pair(sf + 4 * c, make_sf_desc(src + 512 * c));
            }
            __syncwarp();
          }
        }
        ok = all_ok(mbar_wait_bounded(&full[stage], phase, abort_flag, limit));
        if (!ok) break;
        if constexpr (!MX) {
          // last, since it is what the MMAs wait for
          ok = all_ok(mbar_wait_bounded(&my_tempty[buf], bphase ^ 1u, abort_flag, limit));
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + uint32_t(buf * C::kBN + half * C::kN);
        // descriptors of the stage's tiles; 32 bytes further along K are 2 units
        const uint64_t a0 = desc_a + uint32_t(stage * (kABytes / 16));
        const uint64_t b0 = desc_b + uint32_t(stage * (C::kBBytes / 16));
        if constexpr (MX) {
          const uint32_t idesc = idesc_sf_ids(make_idesc_mx(256, C::kBN), uint32_t(kb & 3));
          const bool slot_end = kb + 1 == kbs || (kb + 1) % (4 * C::kQuads) == 0;
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_mx_pair(d, a0 + 2 * kk, b0 + 2 * kk, idesc, sf, sf + 4,
                             (kb > 0 || kk > 0) ? 1u : 0u);
            tc_commit_pair(&empty[stage]);
            if (slot_end) tc_commit_pair(&sempty[slot]);
          }
          __syncwarp();
          if (slot_end) {
            if (++slot == C::kSfSlots) {
              slot = 0;
              sphase ^= 1u;
            }
          }
        } else {
          constexpr uint32_t idesc = make_idesc(1u, 0u, 256, C::kN);
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_f8_pair(d, a0 + 2 * kk, b0 + 2 * kk, idesc, kk > 0 ? 1u : 0u);
            tc_commit_pair(&my_tfull[buf]);
            tc_commit_pair(&empty[stage]);
          }
          __syncwarp();
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
        if (leader) tc_commit_pair(&my_tfull[buf]);
        __syncwarp();
        if (++buf == NB) {
          buf = 0;
          bphase ^= 1u;
        }
      }
    }
    if (leader)
      asm volatile(
          "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
              smem_u32(final_bar))
          : "memory");
    volatile int no_abort = 0;
    mbar_wait_bounded(final_bar, 0, &no_abort, limit);
  } else if (MX && warp == 2) {
    // ---------------- scales: this CTA's tokens, all of the tile's weights ----------------
    const uint8_t* xs = static_cast<const uint8_t*>(p.xs);
    const bool words = kbs >= 4 && p.xs_blk == 1 && p.xs_row % 4 == 0 &&
                       (reinterpret_cast<uintptr_t>(xs) & 3) == 0;
    const int64_t w_blocks = (p.N + 127) / 128;
    const int quads = (kbs + 3) / 4;
    constexpr int Q = C::kQuads;
    ScaleWords<Q> xw;
    BlockWords<Q> ww[C::kSfbChunks];
    auto fetch = [&](int i, int q0) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      xw.fetch(xs, p.xs_row, p.xs_blk, words, int64_t(tile.t) * 256 + rank * kLanes, p.T, lane, q0,
               kbs);
#pragma unroll
      for (int c = 0; c < C::kSfbChunks; ++c) {
        const int64_t nb = int64_t(tile.n) * C::kSfbChunks + c;
        ww[c].fetch(static_cast<const uint8_t*>(p.ws) + nb * kbs, nb < w_blocks, lane, q0, kbs);
      }
    };
    int slot = 0;
    uint32_t sphase = 0;
    bool ok = true;
    Filled filled;
    if (first < tiles) fetch(first, 0);
    for (int i = first; ok && i < tiles; i += step) {
      for (int q0 = 0; q0 < quads; q0 += Q) {
        ok = all_ok(mbar_wait_bounded(&sempty[slot], sphase ^ 1u, abort_flag, limit));
        if (!ok) break;
        uint8_t* dst = sRing + slot * Q * C::kQuadBytes;
        xw.store(dst, C::kQuadBytes, lane);
#pragma unroll
        for (int c = 0; c < C::kSfbChunks; ++c)
          ww[c].store(dst + 512 * (1 + c), C::kQuadBytes, lane);
        // the copies to tensor memory read it through the async proxy
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(peer_addr(smem_u32(&sfull[slot]), 0));
        filled.add(slot, sphase);
        // the next words' loads run while the slots ahead are used
        if (q0 + Q < quads)
          fetch(i, q0 + Q);
        else if (i + step < tiles)
          fetch(i + step, 0);
        if (++slot == C::kSfSlots) {
          slot = 0;
          sphase ^= 1u;
        }
      }
    }
    filled.released(sempty, C::kSfSlots, abort_flag, limit);
  } else if (warp >= 4) {
    // ---------------- promotion and epilogue of this CTA's 128 tokens ----------------
    if constexpr (!MX) setmaxnreg_inc<C::kEpiRegs>();
    const int row = (warp & 3) * 32 + lane;
    const int col0 = ((warp - 4) >> 2) * COLS;
    const uint32_t lane_base = tmem_base + (uint32_t((warp & 3) * 32) << 16) + uint32_t(col0);
    uint64_t* const my_tfull = tfull + (C::kHalves == 1 ? 0 : col0 / C::kN) * NB;
    const uint32_t my_tempty =
        peer_addr(smem_u32(tempty + (C::kHalves == 1 ? 0 : col0 / C::kN) * NB), 0);
    const int64_t w_blocks = (p.N + 127) / 128;
    constexpr int kVec = 16 / int(sizeof(TOUT));
    int buf = 0;
    uint32_t bphase = 0;
    bool ok = true;
    for (int i = first; ok && i < tiles; i += step) {
      const Tile tile = tile_at(i, p.t_tiles, p.n_tiles);
      const int64_t t = int64_t(tile.t) * 256 + rank * kLanes + row;
      const int64_t n0 = int64_t(tile.n) * C::kBN + col0;
      if (p.add != nullptr && t < p.T) {
        // this row's addend is in L2 by the time its sums are done
        const TOUT* add = static_cast<const TOUT*>(p.add) + t * p.ld_add + n0;
#pragma unroll
        for (int j = 0; j < COLS; j += 128 / int(sizeof(TOUT)))
          if (n0 + j < p.N) l2_prefetch(add + j);
      }
      float acc[COLS];
      if constexpr (MX) {
        ok = mbar_wait_bounded(&my_tfull[buf], bphase, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t v[COLS];
        tmem_ld32(lane_base + uint32_t(buf * C::kBN), *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld32(lane_base + uint32_t(buf * C::kBN) + 32,
                  *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tmem_arrived(v);
#pragma unroll
        for (int j = 0; j < COLS; ++j) acc[j] = __uint_as_float(v[j]);
        // the tile is in registers: the next one's MMAs may start
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_read(my_tempty + 8 * buf);
        if (++buf == NB) {
          buf = 0;
          bphase ^= 1u;
        }
      } else {
        const int64_t wb = min(n0 / 128, w_blocks - 1);  // columns past N have no scale
        const float* sx = static_cast<const float*>(p.xs) + (t < p.T ? t * p.xs_row : 0);
        const float* sw = static_cast<const float*>(p.ws) + wb * kbs;
#pragma unroll
        for (int j = 0; j < COLS; ++j) acc[j] = 0.0f;
        // the next k-block's scales are on their way while this one is added
        float s = __ldg(sx) * __ldg(sw);
        for (int kb = 0; kb < kbs; ++kb) {
          ok = all_ok(mbar_wait_bounded(&my_tfull[buf], bphase, abort_flag, limit));
          if (!ok) break;
          tc_fence_after();
          const uint32_t base = lane_base + uint32_t(buf * C::kBN);
          // four batches of 32 columns, the third and fourth on their way while
          // the first two are added
          uint32_t v[2][32];
          tmem_ld32(base, v[0]);
          tmem_ld32(base + 32, v[1]);
          tmem_ld_wait();
          asm volatile("" : "+f"(s));  // no product can move before the wait
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              acc[32 * c + j] = fmaf(s, __uint_as_float(v[c][j]), acc[32 * c + j]);
            tmem_ld32(base + 64 + 32 * c, v[c]);
          }
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_read(my_tempty + 8 * buf);
          float s2 = s;
          asm volatile("" : "+f"(s2));
          if (kb + 1 < kbs) {
            sx += p.xs_blk;
            ++sw;
            s = __ldg(sx) * __ldg(sw);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              acc[64 + 32 * c + j] = fmaf(s2, __uint_as_float(v[c][j]), acc[64 + 32 * c + j]);
          if (++buf == NB) {
            buf = 0;
            bphase ^= 1u;
          }
        }
        if (!ok) break;
      }
      TOUT* out = static_cast<TOUT*>(p.out) + n0;
      const TOUT* add = static_cast<const TOUT*>(p.add) + n0;
      if constexpr (!VEC) {
        // A row's 64 bytes go to memory as elements of neighbouring lanes.
        constexpr int kRun = C::kRunBytes / int(sizeof(TOUT));
        constexpr int kPitch = C::kPitchBytes / int(sizeof(TOUT));
        TOUT* const piece = reinterpret_cast<TOUT*>(sOut + (warp - 4) * C::kStageOut);
        const int64_t t32 = t - lane;
        const int c = lane % kRun;
#pragma unroll
        for (int j = 0; j < COLS; j += kRun) {
          if (n0 + j >= p.N) break;
          const bool in = n0 + j + c < p.N;
          if (p.add != nullptr) {
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += 32 / kRun) {
              const int r = r0 + lane / kRun;
              piece[r * kPitch + c] =
                  in && t32 + r < p.T ? add[(t32 + r) * p.ld_add + j + c] : from_f32<TOUT>(0.0f);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < kRun; ++k) acc[j + k] += to_f32(piece[lane * kPitch + k]);
          }
          uint32_t* const words = reinterpret_cast<uint32_t*>(piece + lane * kPitch);
#pragma unroll
          for (int h = 0; h < C::kRunBytes / 16; ++h) {
            const uint4 v = pack16<TOUT>(&acc[j + h * kVec]);
            words[4 * h] = v.x;
            words[4 * h + 1] = v.y;
            words[4 * h + 2] = v.z;
            words[4 * h + 3] = v.w;
          }
          __syncwarp();
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 32 / kRun) {
            const int r = r0 + lane / kRun;
            if (in && t32 + r < p.T) out[(t32 + r) * p.ld_out + j + c] = piece[r * kPitch + c];
          }
          __syncwarp();
        }
      } else {
        // N is a multiple of kVec. A quad of lanes trades vectors so that it
        // stores 64 bytes of one row at a time (and reads the addend so).
        const int64_t t4 = t - (lane & 3);
        const int mine = (lane & 3) * kVec;
#pragma unroll
        for (int j = 0; j < COLS; j += 4 * kVec) {
          const bool in = n0 + j + mine < p.N;
          uint4 v[4];
          if (p.add != nullptr) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              v[r] = in && t4 + r < p.T
                         ? *reinterpret_cast<const uint4*>(add + (t4 + r) * p.ld_add + j + mine)
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
            if (in && t4 + r < p.T)
              *reinterpret_cast<uint4*>(out + (t4 + r) * p.ld_out + j + mine) = v[r];
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_sync();  // the even CTA's MMAs read both CTAs' memory until here
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(512)
                 : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) report_status(p.status, MOE_ERR_TIMEOUT);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Plan {
  int pair;    // 1: fp8_pair_kernel
  int bn;      // columns per tile (tokens; weight rows for fp8_pair_kernel)
  int splits;  // CTAs per cluster along K
  int ctas;
};

// Nanoseconds by a model whose constants were fitted to the measured times of
// every plan at 51 products (T 1 to 4096, N 512 to 36864, K 300 to 18432): the
// tiles that an SM takes one after another, each its k-blocks and its epilogue.
// What a k-block costs is the way through the ring (kb, kb_col) or, with two
// CTAs on an SM, the bytes and columns of both (share, share_col). Its choice
// was 1.02 times the best plan's time on average and 1.2 times at worst.
struct PlanCost {
  float kb, kb_col, share, share_col, tile, tile_col, split, split_col, pair_kb, pair_tile;
};
constexpr PlanCost kCost[2] = {
    {250, 1.7, 150, 2.5, 450, 8, 1250, 20, 580, 2400},  // fp32 scales
    {265, 0.3, 170, 0.4, 0, 15, 1100, 28, 275, 3400}};  // UE8M0

// Both sides measured, UE8M0, one B200, back to back: 16 x 4096 x 7168 in 8
// pieces 9.4 us, in 4 9.5, unsplit 17.4; 128 x 7168 x 2048 in tiles of 32 tokens 8.7 us,
// of 128 9.2, of 128 in two pieces 13.4; 512 x 4096 x 7168 as pairs 21.9 us (which
// the model takes), in tiles of 128 21.4; 1024 x 4096 x 7168 24.5 and 37.6. fp32
// scales: 512 x 4096 x 7168 as pairs 37.1 us, in tiles of 128 28.8; 1024 x 4096 x
// 7168 38.8 and 55.2.
// In 32 bits, which check_sizes allows, and by shifts: a call makes a plan.
Plan plan_matmul(int64_t T, int64_t N, int64_t K, bool mx, int sms) {
  const uint32_t tokens = uint32_t(T), blocks = uint32_t(ceil_div(N, kLanes));
  const uint32_t kbs = uint32_t(ceil_div(K, kKB)), all = uint32_t(sms);
  const PlanCost& c = kCost[mx];
  Plan best = {0, 16, 1, 1};
  float best_cost = INFINITY;
  for (int lb = 4; lb <= (mx ? 8 : 7); ++lb) {
    const uint32_t bn = 1u << lb;
    if (lb > 4 && bn / 2 >= tokens) break;  // the half would hold every token
    const uint32_t tiles = ((tokens + bn - 1) >> lb) * blocks;
    const uint32_t occ = bn <= 64 ? 2 : 1;
    // clusters of other sizes leave SMs idle: 16 x 7168 x 18432 in 4 pieces
    // 24.5 us, in 5 29.0
    for (int ls = 0; ls <= 3 && (1u << ls) <= kbs; ++ls) {
      const uint32_t ctas = tiles << ls;
      if (ls > 0 && ctas > all * occ) break;
      const uint32_t on_sm = ctas > all ? occ : 1;
      const float rounds = float((ctas + all * on_sm - 1) / (all * on_sm));
      const float kb = std::max(c.kb + c.kb_col * bn, on_sm * (c.share + c.share_col * bn));
      const float cost =
          rounds * (float((kbs + (1u << ls) - 1) >> ls) * kb + c.tile + c.tile_col * bn) +
          (ls > 0 ? c.split + c.split_col * bn : 0.0f);
      if (cost < best_cost) {
        best_cost = cost;
        best = {0, int(bn), 1 << ls, int(std::min(ctas, all * occ))};
      }
    }
  }
  if (tokens > 128) {
    const uint32_t tiles = ((tokens + 255) >> 8) * uint32_t(ceil_div(N, 256));
    const float rounds = float((tiles + all / 2 - 1) / (all / 2));
    if (rounds * (kbs * c.pair_kb + c.pair_tile) < best_cost)
      best = {1, 256, 1, int(2 * std::min(tiles, all / 2))};
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

template <bool MX, bool VEC, typename TOUT>
int launch_pair(const Plan& plan, const CUtensorMap& w, const CUtensorMap& x,
                const MatmulParams& p, cudaStream_t s) {
  using C = PairCfg<MX, VEC>;
  static std::atomic<uint64_t> done{0};
  int st = set_smem_once(fp8_pair_kernel<MX, VEC, TOUT>, C::kSmem, done);
  if (st != MOE_OK) return st;
  // a register split that the launch cannot cover would never return
  static const int regs = [] {
    cudaFuncAttributes attr;
    const cudaError_t e = cudaFuncGetAttributes(&attr, fp8_pair_kernel<MX, VEC, TOUT>);
    return e == cudaSuccess ? attr.numRegs : -1;
  }();
  KSW_REQUIRE(MX || regs == C::kLaunchRegs, MOE_ERR_UNSUPPORTED,
              "fp8_matmul: compiled register count does not match the setmaxnreg split");
  return launch_clusters(fp8_pair_kernel<MX, VEC, TOUT>, plan.ctas, C::kThreads, C::kSmem, 2, s, x,
                         w, p);
}

template <typename TOUT>
int run_matmul(const Plan& plan, bool mx, bool vec, const CUtensorMap& w, const CUtensorMap& x,
               const MatmulParams& p, cudaStream_t s) {
  if (plan.pair && vec)
    return mx ? launch_pair<true, true, TOUT>(plan, w, x, p, s)
              : launch_pair<false, true, TOUT>(plan, w, x, p, s);
  if (plan.pair)
    return mx ? launch_pair<true, false, TOUT>(plan, w, x, p, s)
              : launch_pair<false, false, TOUT>(plan, w, x, p, s);
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
  info[0] = plan.pair;
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
  const int vec = out_dtype == MOE_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  const bool aligned = out_cols % vec == 0 && ld_out % vec == 0 && aligned16(out) &&
                       (addend == nullptr || (ld_addend % vec == 0 && aligned16(addend)));
  const Plan plan = plan_matmul(num_rows, out_cols, inner, mx, sms);
  CUtensorMap tx, tw;
  const uint32_t x_box = plan.pair ? kLanes : uint32_t(plan.bn);
  st = encode_tma_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, uint64_t(inner),
                     uint64_t(num_rows), uint64_t(ld_x), kKB, x_box);
  if (st != MOE_OK) return st;
  const uint32_t pair_box = mx ? PairCfg<true, true>::kBox : PairCfg<false, true>::kBox;
  const uint32_t w_box = plan.pair ? pair_box : kLanes;
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
  p.t_tiles = int(ceil_div(num_rows, plan.pair ? 256 : plan.bn));
  p.n_tiles = int(ceil_div(out_cols, plan.pair ? plan.bn : kLanes));
  p.splits = plan.splits;
  p.slice = int(round_up(ceil_div(plan.bn, plan.splits), 4));
  p.status = status;
  p.wait_limit_ns = kWaitLimitNs;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (out_dtype == MOE_DTYPE_F32) return run_matmul<float>(plan, mx, aligned, tw, tx, p, s);
  if (out_dtype == MOE_DTYPE_BF16)
    return run_matmul<__nv_bfloat16>(plan, mx, aligned, tw, tx, p, s);
  return run_matmul<__half>(plan, mx, aligned, tw, tx, p, s);
}
