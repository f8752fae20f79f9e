// Products of rows in 4 bits on the tensor cores (sm_100a): Y[r] = X[row(r)] W[e]^T over ragged rows, as egs_ragged.cu's, with a scale for every
// block of 32 contraction elements of both operands.  tcgen05.mma kind::mxf4 multiplies the scales in; sums are float32.
//
// Persistent CTAs, or pairs of them, walk tiles of 128 (256) sorted rows of one expert x BN columns.  A step is 256 elements, 128 bytes of a row:
// four MMAs.  Their scales lie in tensor memory beside two accumulators, which leaves 224 columns for each: a tile is no wider.
//
//   warps 0, 1    gathered rows of X (tile::gather4), where they are gathered
//   warp  2       boxes of rows that follow one another and of weights; announces the bytes of a stage
//   warp  3       tensor-memory allocation; copies a step's scales to tensor memory and issues its MMAs, by the leader of a pair for both CTAs; the
//                 second one's tells the leader of scales that are there
//   warps 4..7    scales: of four steps at a time, from rows to the order in which tensor memory takes them
//   warps 8..15   read-out: tensor memory -> rows of the output, in float32, 16 bits or (activated) in 4 bits with their scales
//
// Scales cannot come by TMA: of a row there are 8 bytes a step, and tensor memory wants four bytes of four rows beside one another.  Both CTAs of a pair
// need the scales of all columns.  What the second one's warps have stored and fenced for the async proxy they hand to a warp of their CTA that has nothing on its way, and that
// one hands it over to the leader with a release at cluster scope, which the leader's wait acquires: releases by the storing warps themselves wait
// for the scales that they have asked for behind a memory barrier (94 us for 74 at 8192 x 4096 -> 4096).  Scales word by word with cp.async: 106; 16 bytes of a row (two steps) at a time for 64: 80 for 70.
//
// 8192 x 4096 -> 4096: 66 us, 4.1 PFLOP/s (2.5 times the 16-bit rate; loads alone 47).  No unit is full (tensor pipe 55 %, L2 35 %): waits between the steps,
// 16 pairs of 74 at work in the ninth round of tiles, 4256 columns for 4096.
// 65536 rows of 64 experts, 2048 -> 512: 57, into float32 63, into 4 bits 55 and activated 68; 512 -> 2048, two steps a tile: 82, of which some 30 are the read-out, into float32 129: 268 and 537 MB of
// output (41, 82) share the memory with the loads.  Rows of a block kept in shared memory for all column tiles: 72 for 55; a read-out of both halves at once: no gain.
#include <cstddef>

#include "egs_fp4.cuh"
#include "egs_tcgen05.cuh"

namespace egs {

namespace {

constexpr int kGatherWarps = 2, kBoxWarp = 2, kIssueWarp = 3, kScaleWarp0 = 4, kScaleWarps = 4, kReadWarp0 = 8, kReadWarps = 8;
constexpr int kFp4Threads = (kReadWarp0 + kReadWarps) * 32;
constexpr uint32_t kFp4Header = 512;
constexpr uint32_t kATile = 16384;                 // 128 rows x 128 bytes
constexpr uint32_t kReadArea = 4096;               // transpose of a read-out warp
constexpr size_t kFp4Smem = 227 * 1024;
constexpr int kSmCount = 148;
constexpr int kStepElems = 256, kStepBlocks = 8;
constexpr int kChunkSteps = 4;                     // steps whose scales come together
constexpr uint32_t kAtom = 512;                    // scales of 128 rows and four blocks: [32 rows][4 x 32 rows][4 blocks]
constexpr uint32_t kChunkA = kChunkSteps * 2 * kAtom, kChunkB = 2 * kChunkA, kChunkBytes = kChunkA + kChunkB;
constexpr uint32_t kScaleCols = 24;                // tensor-memory columns of a step's scales: 2 x 4 of rows, 2 x 8 of columns

constexpr int kScaleRing = 2;                      // chunks that are on their way

struct __align__(16) Fp4Header {
  unsigned long long full[kMaxStages];
  unsigned long long empty[kMaxStages];
  unsigned long long scale_full[kScaleRing];
  unsigned long long scale_stored[kScaleRing];       // of the second CTA of a pair, before the leader knows
  unsigned long long scale_empty[kScaleRing];
  unsigned long long acc_full[2];
  unsigned long long acc_empty[2];
  unsigned long long drain;
  uint32_t tmem_base;
  uint32_t abort_flag;
  int warp_sums[kFp4Threads / 32];
};
static_assert(sizeof(Fp4Header) <= kFp4Header, "header does not fit");

struct Fp4Tiles {
  int BN, stages, steps, blocks;
  int tiles_n;
  int gathers;                 // X's rows are gathered
  int vectors, words;          // rows of the output begin on 16 bytes and are whole 16 bytes; of 16-bit elements, on four bytes and whole words
  uint32_t table_bytes;        // of each of the two tables
  Div by_n;
};

template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
  if (PAIR) tma_load_3d_pair(dst, map, x, y, z, bar);
  else tma_load_3d(dst, map, x, y, z, bar);
}
template <bool PAIR>
__device__ __forceinline__ void load_rows4(uint32_t dst, const void* map, int x, const int (&r)[4], uint32_t bar) {
  if (PAIR)
    tma_gather4_pair(dst, map, x, r[0], r[1], r[2], r[3], bar);
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(bar)
        : "memory");
}

// A step: its scales to tensor memory (512 bytes to four columns of all four groups of lanes: those of the rows at sa, of the columns at sa + 8, the second half of the step's
// four and eight columns on), then four contraction steps of 64 elements.  One block of PTX: the warp's own instructions between them cost more than they.
#define EGS_FP4_STEP(GROUP, WIDE)                                                                                   \
  asm volatile(                                                                                                     \
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t.reg .b32 i, s, t, u, v;\n\t"                                     \
      "add.u32 s, %4, 4;\n\tadd.u32 t, %4, 8;\n\tadd.u32 u, %4, 16;\n\tadd.u32 v, %4, 12;\n\t"                       \
      "add.u64 a, %5, 32;\n\tadd.u64 b, %6, 64;\n\t"                                                               \
      "tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [%4], %5;\n\t"                                                \
      "tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [s], a;\n\t"                                                  \
      "tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [t], %6;\n\t"                                                 \
      "tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [u], b;\n\t" WIDE                                             \
      "setp.ne.b32 p, %7, 0;\n\tsetp.eq.b32 q, 0, 0;\n\tor.b32 i, %3, 0x40000020;\n\t"                              \
      "tcgen05.mma.cta_group::" GROUP ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [t], p;\n\t"   \
      "add.u64 a, %1, 2;\n\tadd.u64 b, %2, 2;\n\t"                                                                 \
      "tcgen05.mma.cta_group::" GROUP ".kind::mxf4.block_scale.scale_vec::2X [%0], a, b, i, [%4], [t], q;\n\t"      \
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"                                                                   \
      "tcgen05.mma.cta_group::" GROUP ".kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [s], [u], q;\n\t"      \
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"                                                                   \
      "tcgen05.mma.cta_group::" GROUP ".kind::mxf4.block_scale.scale_vec::2X [%0], a, b, i, [s], [u], q;\n\t}"      \
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa), "l"(from_a), "l"(from_b), "r"(accumulate)         \
      : "memory")
// (more than 128 columns: another 512 bytes for each half)
#define EGS_FP4_WIDE(GROUP)                                            \
  "add.u64 a, %6, 32;\n\tadd.u64 b, %6, 96;\n\t"                      \
  "tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [v], a;\n\t"         \
  "add.u32 v, %4, 20;\n\t"                                            \
  "tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [v], b;\n\t"
template <bool PAIR>
__device__ __forceinline__ void step_fp4(bool wide, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sa, uint64_t from_a, uint64_t from_b, uint32_t accumulate) {
  if (wide) {
    if (PAIR) EGS_FP4_STEP("2", EGS_FP4_WIDE("2"));
    else EGS_FP4_STEP("1", EGS_FP4_WIDE("1"));
  } else {
    if (PAIR) EGS_FP4_STEP("2", "");
    else EGS_FP4_STEP("1", "");
  }
}

struct RingCursor {
  int slot = 0, round = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++slot == stages) {
      slot = 0;
      ++round;
    }
  }
};

// The expert of row block `block`, from the numbers of the blocks before each expert's; `e` is where the last search ended.
__device__ __forceinline__ int expert_of(const int* starts, int E, int block, int e) {
  if (starts[e + 1] > block) return e;
  int lo = e + 1, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid + 1] > block) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// 16 bytes of a row's scales from block `b` on as words; zeros behind the row's end (whose 16 bytes may be read to their end) and for rows that are not there.
__device__ __forceinline__ void load_scales(const uint8_t* row, int b, int blocks, uint32_t (&w)[4]) {
  const uint4 x = row && b < blocks ? *reinterpret_cast<const uint4*>(row + b) : make_uint4(0u, 0u, 0u, 0u);
  w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  if (b + 16 > blocks) {
    const int left = 8 * (blocks - b);               // bits
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= left >= 32 * (i + 1) ? 0xffffffffu : left > 32 * i ? (1u << (left - 32 * i)) - 1u : 0u;
  }
}

// The warps that bring scales.  P neighbouring lanes have 16 P bytes of a row, 16 each, and a lane hands its words over when their two steps come, with four steps'; what is behind is
// asked for `kSets` such stretches ahead.  A request of the L2 takes as long for 16 bytes as for 64: 16 or 32 bytes of a row at a time, scales held up the operands (8192 x
// 4096 -> 4096: 80 us, 64 bytes 70), while stretches longer than a contraction leave nothing on its way under a tile (512 -> 2048: 64 bytes 197 us, 16 86).
struct ScaleTiles {
  const int *offsets, *starts;
  int units, first, stride, block, row0;
  uint32_t scales, stored, empty;      // stored: the barrier of this CTA's warps
  volatile uint32_t* abort_flag;
};
template <int P>
__device__ __forceinline__ void scale_warps(const Fp4Params& p, const Fp4Tiles& q, const ScaleTiles& t) {
  constexpr int kSets = P == 1 ? 3 : P == 2 ? 2 : 1, kTurn = 128 / P, kColTurns = P == 4 ? 7 : 2 * P;      // (a tile has 224 columns at most)
  struct Words {
    uint32_t a[P][4], b[kColTurns][4];
    int chunks;
  };
  const int lane = threadIdx.x & 31, piece = lane % P, mine = (threadIdx.x / 32 - kScaleWarp0) * (32 / P) + lane / P;
  int round = 0, s0 = 0, e = 0;
  int row[P], coming[P], columns_here = 0;           // rows of X of the tile and (their slots) of the next one
  const uint8_t* b_rows = nullptr;
  auto unit_of = [&](int r) { return r * t.stride + t.first; };
  auto rows_of = [&](int u) {
    if (u >= t.units) return;
    const int block = q.by_n.quotient(u);
    e = expert_of(t.starts, p.E, block, e);
    const int r = t.offsets[e] + (block - t.starts[e]) * t.block + t.row0 + mine, end = t.offsets[e + 1];
#pragma unroll
    for (int i = 0; i < P; ++i) coming[i] = r + i * kTurn < end ? p.slots ? p.slots[r + i * kTurn] : r + i * kTurn : -1;
  };
  auto ask = [&](Words& w) {
    const int u = unit_of(round);
    w.chunks = 0;
    if (u >= t.units) return;
    if (s0 == 0) {
      const int block = q.by_n.quotient(u), n0 = (u - block * q.tiles_n) * q.BN;
      columns_here = min(q.BN, p.N - n0);
#pragma unroll
      for (int i = 0; i < P; ++i) row[i] = coming[i] >= 0 && p.slots ? p.by_k.quotient(coming[i]) : coming[i];
      b_rows = p.Ws + e * p.ws_expert + (n0 + mine) * p.ws_row;
      rows_of(unit_of(round + 1));
    }
    const int first = s0 * kStepBlocks + piece * 16;
#pragma unroll
    for (int i = 0; i < P; ++i) load_scales(row[i] >= 0 ? p.As + row[i] * p.as_row : nullptr, first, q.blocks, w.a[i]);
#pragma unroll
    for (int i = 0; i < kColTurns; ++i) load_scales(mine + i * kTurn < columns_here ? b_rows + i * kTurn * p.ws_row : nullptr, first, q.blocks, w.b[i]);
    w.chunks = min((P + 1) / 2, (q.steps - s0 + kChunkSteps - 1) / kChunkSteps);
    s0 += 2 * P;
    if (s0 >= q.steps) {
      s0 = 0;
      ++round;
    }
  };
  RingCursor chunk;
  auto turn = [&](Words& w) {
    if (w.chunks == 0) return false;
#pragma unroll 1
    for (int c = 0; c < w.chunks; ++c) {
      if (chunk.round > 0 && !mbar_wait_all(t.empty + chunk.slot * 8u, (chunk.round - 1) & 1, t.abort_flag, p.status.word)) return false;
      if (piece >> 1 == c) {
        const uint32_t to = t.scales + static_cast<uint32_t>(chunk.slot) * kChunkBytes, half = static_cast<uint32_t>(piece & 1) * 4u;      // (four words of a chunk's eight)
        auto put = [&](uint32_t base, uint32_t stride, int r, const uint32_t (&x)[4]) {
          const uint32_t at = base + static_cast<uint32_t>(r & 31) * 16u + static_cast<uint32_t>(r >> 5 & 3) * 4u;
#pragma unroll
          for (int j = 0; j < 4; ++j) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + static_cast<uint32_t>(j) * stride), "r"(x[j]) : "memory");
        };
#pragma unroll
        for (int i = 0; i < P; ++i) put(to + half * kAtom, kAtom, i * kTurn + mine, w.a[i]);
#pragma unroll
        for (int i = 0; i < kColTurns; ++i) put(to + kChunkA + (half * 2u + static_cast<uint32_t>(i * kTurn >> 7)) * kAtom, 2u * kAtom, i * kTurn + mine, w.b[i]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(t.stored + chunk.slot * 8u);
      chunk.next(kScaleRing);
    }
    ask(w);
    return true;
  };
  Words w[kSets];
  rows_of(unit_of(0));
#pragma unroll
  for (int i = 0; i < kSets; ++i) ask(w[i]);
  bool more = true;
  while (more) {
#pragma unroll
    for (int i = 0; i < kSets; ++i) more = more && turn(w[i]);
  }
}

struct Fp4Out {};              // rows of the output in 4 bits
template <typename OutT> __device__ __forceinline__ uint32_t pack_out(uint32_t a, uint32_t b) { return pack2(static_cast<OutT*>(nullptr), a, b); }

template <typename OutT, bool PAIR>
__global__ void __cluster_dims__(PAIR ? 2 : 1, 1, 1) __launch_bounds__(kFp4Threads, 1)
fp4_rows_kernel(const __grid_constant__ Fp4Params p, const __grid_constant__ Fp4Tiles q, const __grid_constant__ TensorMap3 map_a,
                const __grid_constant__ TensorMap3 map_a4, const __grid_constant__ TensorMap3 map_b) {
  constexpr bool kFp4Out = std::is_same<OutT, Fp4Out>::value;
  constexpr int kBlock = PAIR ? 256 : 128;           // rows of a tile
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Fp4Header* hdr = reinterpret_cast<Fp4Header*>(smem_raw);
  int* offsets = reinterpret_cast<int*>(smem_raw + kFp4Header);
  int* starts = reinterpret_cast<int*>(smem_raw + kFp4Header + q.table_bytes);      // row blocks before each expert's
  const uint32_t smem0 = smem_u32(smem_raw);
  const uint32_t ring0 = (smem0 + kFp4Header + 2u * q.table_bytes + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? static_cast<int>(blockIdx.x & 1) : 0;
  const bool leader = rank == 0;
  const int columns = PAIR ? q.BN / 2 : q.BN;        // of the right operand, staged by this CTA
  const uint32_t stage_bytes = kATile + static_cast<uint32_t>(columns) * 128u;
  const uint32_t scales0 = ring0 + static_cast<uint32_t>(q.stages) * stage_bytes;      // (rows of 128 bytes, eight at a time: whole 1024 bytes)
  const uint32_t area0 = scales0 + kScaleRing * kChunkBytes;                 // (rows in 4 bits need none)
  const uint32_t acc_cols = static_cast<uint32_t>(q.BN), scale_cols = 2u * acc_cols, all_cols = tmem_cols_for(2 * q.BN + 2 * static_cast<int>(kScaleCols));
  volatile uint32_t* abort_flag = &hdr->abort_flag;
  const int first_unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, unit_stride = PAIR ? gridDim.x >> 1 : gridDim.x;

  // ---- set-up ----
  if (tid == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(smem_u32(&hdr->full[s]), 1);
      mbar_init(smem_u32(&hdr->empty[s]), 1);
    }
    for (int b = 0; b < kScaleRing; ++b) {
      mbar_init(smem_u32(&hdr->scale_full[b]), PAIR ? kScaleWarps + 1 : kScaleWarps);  // (a pair's: the leader's copy is used)
      mbar_init(smem_u32(&hdr->scale_stored[b]), kScaleWarps);
      mbar_init(smem_u32(&hdr->scale_empty[b]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&hdr->acc_full[b]), 1);
      mbar_init(smem_u32(&hdr->acc_empty[b]), PAIR ? 2 * kReadWarps : kReadWarps);     // (the leader's too)
    }
    mbar_init(smem_u32(&hdr->drain), 1);
    fence_mbar_init();
  }
  pdl_wait();
  if (tid == 0) {
    hdr->abort_flag = p.status.timed_out() ? 1u : 0u;
    if (smem_misaligned(smem_raw)) {
      hdr->abort_flag = 1u;
      p.status.report(EGS_STATUS_INTERNAL);
    }
  }
  if (p.offsets)
    for (int e = tid; e <= p.E; e += kFp4Threads) offsets[e] = p.offsets[e];
  else if (tid < 2)
    offsets[tid] = tid ? p.rows : 0;
  __syncthreads();
  if (warp == kIssueWarp) {
    if (PAIR) {
      tmem_alloc2(smem_u32(&hdr->tmem_base), all_cols);
      tmem_relinquish2();
    } else {
      tmem_alloc(smem_u32(&hdr->tmem_base), all_cols);
      tmem_relinquish();
    }
  }
  for (int e0 = 0, carry = 0; e0 < p.E; e0 += kFp4Threads) {
    const int e = e0 + tid, own = e < p.E ? (offsets[e + 1] - offsets[e] + kBlock - 1) / kBlock : 0;
    int at = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) hdr->warp_sums[warp] = at;
    __syncthreads();
    int before = carry, total = 0;
    for (int w = 0; w < kFp4Threads / 32; ++w) {
      if (w < warp) before += hdr->warp_sums[w];
      total += hdr->warp_sums[w];
    }
    if (e < p.E) starts[e] = at + before - own;
    carry += total;
    if (e == p.E - 1) starts[p.E] = carry;
    __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();                      // both CTAs' barriers are initialised before anything crosses the pair
  tc_fence_after();
  const uint32_t tmem_base = hdr->tmem_base;
  const int units = starts[p.E] * q.tiles_n;
  const uint32_t full0 = PAIR ? map_to_cta(smem_u32(&hdr->full[0]), 0) : smem_u32(&hdr->full[0]);
  auto unit_of = [&](int round) { return round * unit_stride + first_unit; };
  RingCursor at;
  bool alive = true;
  auto wait_free = [&]() {
    if (at.round > 0) alive = mbar_wait_all(smem_u32(&hdr->empty[at.slot]), (at.round - 1) & 1, abort_flag, p.status.word);
    return alive;
  };

  if (hdr->abort_flag != 0u) {
    // fall through to the common exit
  } else if (warp < kGatherWarps) {
    // =========================== gathered rows ===========================
    if (q.gathers) {
      int e = 0;
      for (int round = 0, u; (u = unit_of(round)) < units && alive; ++round) {
        const int block = q.by_n.quotient(u);
        e = expert_of(starts, p.E, block, e);
        const int r = offsets[e] + (block - starts[e]) * kBlock + rank * 128 + warp * 64 + lane, end = offsets[e + 1];
        const int low = r < end ? p.by_k.quotient(p.slots[r]) : -1, high = r + 32 < end ? p.by_k.quotient(p.slots[r + 32]) : -1;
        int row[16][4];
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) row[i][j] = __shfl_sync(0xffffffffu, i < 8 ? low : high, i % 8 * 4 + j);
        for (int ks = 0; ks < q.steps; ++ks) {
          if (!wait_free()) break;
          const uint32_t bar = full0 + at.slot * 8u;
          const uint32_t dst = ring0 + static_cast<uint32_t>(at.slot) * stage_bytes + static_cast<uint32_t>(warp) * 8192u;
          at.next(q.stages);
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < 16; ++i) load_rows4<PAIR>(dst + i * 512u, &map_a4, ks * 128, row[i], bar);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == kBoxWarp) {
    // =========================== boxes ===========================
    const uint32_t bytes = PAIR ? 2u * stage_bytes : stage_bytes;       // announced by the leader for both CTAs
    int e = 0;
    for (int round = 0, u; (u = unit_of(round)) < units && alive; ++round) {
      const int x = q.by_n.quotient(u);
      const int n0 = (u - x * q.tiles_n) * q.BN + rank * columns;
      e = expert_of(starts, p.E, x, e);
      const int a0 = offsets[e] + (x - starts[e]) * kBlock + rank * 128;
      for (int ks = 0; ks < q.steps; ++ks) {
        if (!wait_free()) break;
        const uint32_t own = smem_u32(&hdr->full[at.slot]), bar = full0 + at.slot * 8u;
        const uint32_t a_dst = ring0 + static_cast<uint32_t>(at.slot) * stage_bytes, b_dst = a_dst + kATile;
        at.next(q.stages);
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(own, bytes);
          if (!q.gathers) load_box<PAIR>(a_dst, &map_a, ks * 128, a0, 0, bar);
          load_box<PAIR>(b_dst, &map_b, ks * 128, n0, e, bar);
        }
      }
    }
    __syncwarp();
  } else if (warp == kIssueWarp) {
    // =========================== MMA issuer ===========================
    if (leader) {
      const uint64_t a_desc = make_smem_desc(0u, 16u, 1024u), s_desc = make_smem_desc(0u, 16u, 128u, 0u);
      // E2M1 operands (format 1), scales as powers of two, K-major; places of the scales' bytes come with the MMAs
      const uint32_t idesc = (1u << 7) | (1u << 10) | (static_cast<uint32_t>(q.BN >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(kBlock >> 4) << 24);
      const bool wide = q.BN > 128;
      // What a step needs moves on by additions: multiplications and remainders between two steps' MMAs left the tensor cores waiting.
      int t = 0;
      RingCursor chunk;
      uint32_t parity = 0u;
      const uint32_t sa0 = tmem_base + scale_cols;
      const uint64_t b_far = static_cast<uint64_t>(kATile >> 4), stage_units = static_cast<uint64_t>(stage_bytes >> 4);
      const uint64_t a_first = a_desc + (ring0 >> 4);
      uint64_t a_now = a_first;
      uint32_t full = smem_u32(&hdr->full[0]);
      constexpr uint32_t kEmptyFar = static_cast<uint32_t>(offsetof(Fp4Header, empty) - offsetof(Fp4Header, full));
      for (int round = 0, u; (u = unit_of(round)) < units && alive; ++round) {
        const int buf = t & 1;
        if (t >= 2) {
          alive = mbar_wait_all<PAIR>(smem_u32(&hdr->acc_empty[buf]), ((t >> 1) - 1) & 1, abort_flag, p.status.word);
          if (!alive) break;
        }
        ++t;
        const uint32_t d = tmem_base + static_cast<uint32_t>(buf) * acc_cols;
        for (int ks = 0; ks < q.steps && alive;) {
          const uint32_t scale_full = smem_u32(&hdr->scale_full[chunk.slot]), scale_empty = smem_u32(&hdr->scale_empty[chunk.slot]);
          const uint32_t scales = (scales0 + static_cast<uint32_t>(chunk.slot) * kChunkBytes) >> 4;
          uint64_t from_a = s_desc + scales, from_b = s_desc + scales + (kChunkA >> 4);
          alive = mbar_wait_all<PAIR>(scale_full, chunk.round & 1, abort_flag, p.status.word);
          const int end = min(q.steps, ks + kChunkSteps);
          for (; ks < end && alive; ++ks) {
            alive = mbar_wait_all<PAIR>(full, at.round & 1, abort_flag, p.status.word);
            if (!alive) break;
            tc_fence_after();
            if (elect_one()) {
              step_fp4<PAIR>(wide, d, a_now, a_now + b_far, idesc, sa0 + parity, from_a, from_b, ks > 0 ? 1u : 0u);
              umma_done<PAIR>(full + kEmptyFar);
              if (ks + 1 == end) umma_done<PAIR>(scale_empty);
              if (ks + 1 == q.steps) umma_done<PAIR>(smem_u32(&hdr->acc_full[buf]));
            }
            parity ^= kScaleCols;
            from_a += 2u * kAtom >> 4;
            from_b += 4u * kAtom >> 4;
            a_now += stage_units;
            full += 8u;
            if (++at.slot == q.stages) {
              at.slot = 0;
              ++at.round;
              a_now = a_first;
              full = smem_u32(&hdr->full[0]);
            }
          }
          chunk.next(kScaleRing);
        }
      }
    } else {
      // scales that this CTA's warps have stored: what the wait has acquired of them the arrival releases to the leader
      RingCursor chunk;
      for (int round = 0; unit_of(round) < units && alive; ++round)
        for (int ks = 0; ks < q.steps && alive; ks += kChunkSteps) {
          alive = mbar_wait_all(smem_u32(&hdr->scale_stored[chunk.slot]), chunk.round & 1, abort_flag, p.status.word);
          if (alive && elect_one()) mbar_arrive_cluster(map_to_cta(smem_u32(&hdr->scale_full[chunk.slot]), 0));
          chunk.next(kScaleRing);
        }
    }
    pdl_trigger();
    __syncwarp();
  } else if (warp < kReadWarp0) {
    // =========================== scales ===========================
    const ScaleTiles tiles{offsets, starts, units, first_unit, unit_stride, kBlock, rank * 128, scales0, smem_u32(leader ? &hdr->scale_full[0] : &hdr->scale_stored[0]), smem_u32(&hdr->scale_empty[0]), abort_flag};
    if (q.steps > 4) scale_warps<4>(p, q, tiles);
    else if (q.steps > 2) scale_warps<2>(p, q, tiles);
    else scale_warps<1>(p, q, tiles);
    __syncwarp();
  } else {
    // =========================== read-out ===========================
    const int ew = warp - kReadWarp0, lg = ew & 3, share = ew >> 2;     // TMEM lane group (warp number mod 4), share of the column blocks
    const uint32_t area = area0 + static_cast<uint32_t>(ew) * kReadArea;
    const uint32_t lane_base = static_cast<uint32_t>(lg * 32) << 16;
    if (p.offsets) {                                 // rows that belong to no expert
      const long long routed = offsets[p.E], turn = static_cast<long long>(gridDim.x) * (kReadWarps * 32);
      const long long first = static_cast<long long>(blockIdx.x) * (kReadWarps * 32) + ew * 32 + lane;
      if constexpr (kFp4Out) {
        for (long long r = routed + first; r < p.rows; r += turn)
          for (int i = 0; i < fp4_blocks(p.N); ++i) {
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.Out) + r * p.y_row + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            p.OutScale[r * p.ys_row + i] = 0;
          }
      } else {
        for (long long i = routed * p.N + first; i < static_cast<long long>(p.rows) * p.N; i += turn) static_cast<OutT*>(p.Out)[i] = from_f32<OutT>(0.f);
      }
    }
    int t = 0, e = 0;
    for (int round = 0, u; (u = unit_of(round)) < units && alive; ++round) {
      const int block = q.by_n.quotient(u), n0 = (u - block * q.tiles_n) * q.BN, bn = min(q.BN, p.N - n0);
      e = expert_of(starts, p.E, block, e);
      const int r = offsets[e] + (block - starts[e]) * kBlock + rank * 128 + lg * 32;
      const long long row0 = r;
      const int rows = min(32, offsets[e + 1] - r);
      const int buf = t & 1;
      alive = mbar_wait_all(smem_u32(&hdr->acc_full[buf]), (t >> 1) & 1, abort_flag, p.status.word);
      if (!alive) break;
      ++t;
      tc_fence_after();
      const uint32_t acc = tmem_base + lane_base + static_cast<uint32_t>(buf) * acc_cols;
      bool released = false;
      auto release = [&]() {
        if (released) return;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&hdr->acc_empty[buf]), 0));
          else mbar_arrive(smem_u32(&hdr->acc_empty[buf]));
        }
        released = true;
      };
      if constexpr (kFp4Out) {
        // a lane has a row's 32 columns: a block
        for (int c = share * 32; c < bn; c += 64) {
          uint32_t v[32];
          tmem_ld32(acc + static_cast<uint32_t>(c), v);
          tmem_ld_wait();
          if (c + 64 >= bn) release();
          uint32_t top = 0u;
          if (p.act == EGS_ACT_SILU) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(silu_near(__uint_as_float(v[i])));
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) top = max(top, v[i] & 0x7fffffffu);
          const uint32_t byte = fp4_scale(top);
          const float inverse = fp4_inverse(byte);
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = fp4_scaled(__uint_as_float(v[8 * i + j]), inverse);
            w[i] = fp4_pack8(x);
          }
          if (lane < rows) {
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.Out) + (row0 + lane) * p.y_row + (n0 + c) / 2) = make_uint4(w[0], w[1], w[2], w[3]);
            p.OutScale[(row0 + lane) * p.ys_row + (n0 + c) / kFp4Block] = static_cast<uint8_t>(byte);
          }
        }
      } else if constexpr (sizeof(OutT) == 2) {
        // 64 columns = 128 bytes of a row at a time, eight lanes to a row
        OutT* out = static_cast<OutT*>(p.Out);
        for (int c = share * 64; c < bn; c += 128) {
          const uint32_t srow = area + static_cast<uint32_t>(lane) * 128u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (c + h * 32 < bn) {
              uint32_t v[32];
              tmem_ld32(acc + static_cast<uint32_t>(c + h * 32), v);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 4; ++j)
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(srow + static_cast<uint32_t>((h * 4 + j) ^ (lane & 7)) * 16u),
                             "r"(pack_out<OutT>(v[8 * j], v[8 * j + 1])), "r"(pack_out<OutT>(v[8 * j + 2], v[8 * j + 3])),
                             "r"(pack_out<OutT>(v[8 * j + 4], v[8 * j + 5])), "r"(pack_out<OutT>(v[8 * j + 6], v[8 * j + 7]))
                             : "memory");
            }
          }
          if (c + 128 >= bn) release();              // the accumulator has been read: the next tile but one may begin
          __syncwarp();
          if (q.vectors) {
            const int j = lane & 7, col = c + j * 8;
            uint4 y[8];
#pragma unroll
            for (int it = 0; it < 8; ++it) {
              const int row = it * 4 + (lane >> 3);
              asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(y[it].x), "=r"(y[it].y), "=r"(y[it].z), "=r"(y[it].w)
                           : "r"(area + row * 128u + (static_cast<uint32_t>(j ^ (row & 7)) << 4))
                           : "memory");
            }
#pragma unroll
            for (int it = 0; it < 8; ++it) {
              const int row = it * 4 + (lane >> 3);
              if (row < rows && col < bn) *reinterpret_cast<uint4*>(out + (row0 + row) * p.N + n0 + col) = y[it];
            }
          } else if (q.words) {                      // rows of whole words: a row at a time
            const int col = c + lane * 2;
            OutT* o = out + row0 * p.N + n0 + col;
#pragma unroll 8
            for (int row = 0; row < min(rows, 32); ++row) {
              uint32_t y;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(y) : "r"(area + row * 128u + (static_cast<uint32_t>((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4u) : "memory");
              if (col < bn) *reinterpret_cast<uint32_t*>(o + static_cast<long long>(row) * p.N) = y;
            }
          } else {                                   // rows that begin anywhere: element by element along a row
            for (int row = 0; row < min(rows, 32); ++row)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int i = h * 32 + lane;
                unsigned short b;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(b) : "r"(area + row * 128u + (static_cast<uint32_t>((i >> 3) ^ (row & 7)) << 4) + (i & 7) * 2u) : "memory");
                if (c + i < bn) reinterpret_cast<unsigned short*>(out)[(row0 + row) * p.N + n0 + c + i] = b;
              }
          }
          __syncwarp();
        }
      } else {
        float* out = static_cast<float*>(p.Out);
        for (int c = share * 32; c < bn; c += 64) {
          uint32_t v[32];
          tmem_ld32(acc + static_cast<uint32_t>(c), v);
          tmem_ld_wait();
          if (c + 64 >= bn) release();
          warp_regs_emit(v, area, lane, [&](int row, int cj, uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
            const int col = c + cj;
            if (row >= rows || col >= bn) return;
            float* o = out + (row0 + row) * p.N + n0 + col;
            if (q.vectors) {
              store4(o, x0, x1, x2, x3);
            } else {
              o[0] = __uint_as_float(x0);
              if (col + 1 < bn) o[1] = __uint_as_float(x1);
              if (col + 2 < bn) o[2] = __uint_as_float(x2);
              if (col + 3 < bn) o[3] = __uint_as_float(x3);
            }
          });
        }
      }
      release();                                     // (warps whose share of the columns is empty)
    }
  }

  // ---- common exit (see dense16_kernel) ----
  tc_fence_before();
  __syncthreads();
  if (!PAIR) {
    if (warp == kIssueWarp) tmem_release(tmem_base, all_cols, smem_u32(&hdr->drain), abort_flag, p.status, lane);
  } else {
    uint32_t safe = 1u;
    if (warp == kIssueWarp && *abort_flag) {
      if (lane == 0) {
        uint32_t ignore_abort = 0u;
        p.status.tell_host();
        umma2_commit(smem_u32(&hdr->drain));
        safe = mbar_wait(smem_u32(&hdr->drain), 0u, &ignore_abort, nullptr) ? 1u : 0u;
      }
      safe = __shfl_sync(0xffffffffu, safe, 0);
    }
    cluster_sync_all();
    if (warp == kIssueWarp && safe) {
      tc_fence_after();
      tmem_dealloc2(tmem_base, all_cols);
    }
  }
}

template <typename OutT, bool PAIR>
cudaError_t launch_fp4(const Fp4Params& p, Fp4Tiles q, long long most_units, const TensorMap3 (&maps)[3], cudaStream_t st) {
  q.table_bytes = static_cast<uint32_t>((p.E + 1) * 4 + 15) & ~15u;
  const size_t before = (kFp4Header + 2 * q.table_bytes + 1023u) & ~static_cast<size_t>(1023);
  const size_t stage = kATile + static_cast<size_t>(PAIR ? q.BN / 2 : q.BN) * 128;
  const size_t fixed = before + kScaleRing * kChunkBytes + (std::is_same<OutT, Fp4Out>::value ? 0 : kReadWarps * kReadArea);
  q.stages = static_cast<int>((kFp4Smem - fixed) / stage);
  if (q.stages > kMaxStages) q.stages = kMaxStages;
  cudaError_t err = ensure_smem_optin<fp4_rows_kernel<OutT, PAIR>>(static_cast<int>(kFp4Smem));
  if (err != cudaSuccess) return err;
  const long long workers = PAIR ? kSmCount / 2 : kSmCount;
  const long long grid = (most_units < workers ? (most_units < 1 ? 1 : most_units) : workers) * (PAIR ? 2 : 1);
  count_launch();
  return launch_kernel(fp4_rows_kernel<OutT, PAIR>, static_cast<unsigned>(grid), kFp4Threads, fixed + q.stages * stage, st, true, p, q, maps[0], maps[1], maps[2]);
}
template <typename OutT>
cudaError_t launch_by_pair(const Fp4Params& p, const Fp4Tiles& q, bool pair, long long units, const TensorMap3 (&maps)[3], cudaStream_t st) {
  return pair ? launch_fp4<OutT, true>(p, q, units, maps, st) : launch_fp4<OutT, false>(p, q, units, maps, st);
}

struct TileChoice {
  bool pair;
  int BN;
};
// The tile of least estimated time, as egs_ragged.cu chooses: a step costs its bytes at 60 a clock or its MMAs, two clocks a column.
template <class Blocks>
TileChoice choose_tile(int N, long long steps, Blocks&& blocks) {
  constexpr TileChoice kCandidates[] = {{true, 224}, {false, 224}, {true, 192}, {true, 128}, {false, 128}, {false, 64}};
  TileChoice best{false, 64};
  double least = -1;
  for (const TileChoice& c : kCandidates) {
    const int tiles = (N + c.BN - 1) / c.BN, BN = ((N + tiles - 1) / tiles + 31) / 32 * 32;
    const int workers = c.pair ? kSmCount / 2 : kSmCount;
    const double bytes = kATile + (c.pair ? BN / 2 : BN) * 128.0 + (128 + BN) * 8.0, mma = 2.0 * BN;
    const double work = (bytes / 60 > mma ? bytes / 60 : mma) * steps, out = 1500 + 3500.0 * BN / 256;
    const long long units = static_cast<long long>(blocks(c.pair ? 256 : 128) * tiles);
    const double time = static_cast<double>((units + workers - 1) / workers) * (work > out ? work : out) + out;
    if (least < 0 || time < 0.97 * least) {
      least = time;
      best = {c.pair, BN};
    }
  }
  return best;
}

}  // namespace

cudaError_t launch_fp4_rows_tensor(const Fp4Params& p, int out_dtype, cudaStream_t st) {
  const bool fp4_out = p.OutScale != nullptr;
  const int out_elem = out_dtype == EGS_F32 ? 4 : 2;
  Fp4Tiles q{};
  q.blocks = fp4_blocks(p.C);
  q.steps = (p.C + kStepElems - 1) / kStepElems;
  const int experts = p.offsets ? (p.rows < p.E ? p.rows : p.E) : 1;
  const double each = static_cast<double>(p.rows) / experts;
  // (an expert's last block is half empty in the mean)
  const TileChoice tile = choose_tile(p.N, q.steps, [&](int rows) { return experts * (each <= rows / 2 ? 1.0 : !p.offsets ? (p.rows + rows - 1) / rows : each / rows + 0.5); });
  q.BN = tile.BN;
  q.tiles_n = (p.N + q.BN - 1) / q.BN;
  q.by_n = Div(q.tiles_n);
  q.gathers = p.slots != nullptr;
  const uintptr_t out = reinterpret_cast<uintptr_t>(p.Out);
  q.vectors = (static_cast<long long>(p.N) * out_elem) % 16 == 0 && (out & 15u) == 0;
  q.words = p.N % 2 == 0 && (out & 3u) == 0;
  const int block = tile.pair ? 256 : 128, columns = tile.pair ? q.BN / 2 : q.BN;
  const long long blocks = p.offsets ? p.rows / block + (p.rows < p.E ? p.rows : p.E) : (p.rows + block - 1) / block;
  const unsigned long long width = static_cast<unsigned long long>((p.C + 1) / 2);
  TensorMap3 maps[3];
  {
    const unsigned long long dims[3] = {width, static_cast<unsigned long long>(p.a_rows), 1ull};
    const unsigned long long strides[2] = {static_cast<unsigned long long>(p.a_row), static_cast<unsigned long long>(p.a_row) * p.a_rows};
    const unsigned box[3] = {128u, 128u, 1u}, four[2] = {128u, 1u};
    if (!encode_tensor_map_strided(&maps[0], p.A, 1, 3, dims, strides, box) || !encode_tensor_map_strided(&maps[1], p.A, 1, 2, dims, strides, four))
      return cudaErrorInvalidValue;
  }
  const unsigned long long dims[3] = {width, static_cast<unsigned long long>(p.N), static_cast<unsigned long long>(p.E)};
  const unsigned long long strides[2] = {static_cast<unsigned long long>(p.w_row), static_cast<unsigned long long>(p.w_expert)};
  const unsigned box[3] = {128u, static_cast<unsigned>(columns), 1u};
  if (!encode_tensor_map_strided(&maps[2], p.W, 1, 3, dims, strides, box)) return cudaErrorInvalidValue;
  const long long units = blocks * q.tiles_n;
  if (fp4_out) return launch_by_pair<Fp4Out>(p, q, tile.pair, units, maps, st);
  if (out_dtype == EGS_F16) return launch_by_pair<__half>(p, q, tile.pair, units, maps, st);
  if (out_dtype == EGS_BF16) return launch_by_pair<__nv_bfloat16>(p, q, tile.pair, units, maps, st);
  return launch_by_pair<float>(p, q, tile.pair, units, maps, st);
}

}  // namespace egs
