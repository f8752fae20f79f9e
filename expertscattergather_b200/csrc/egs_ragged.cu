// Products over ragged rows on the tensor cores (sm_100a): the rows of expert e are the sorted rows offsets[e] .. offsets[e + 1] - 1,
// a different number for every expert, known on the device alone.  16-bit operands with float32 sums, 8-bit integers with int32 sums.
//
//   rows      Y[r] = X[row(r)] W[e]            tiles of 128 sorted rows of one expert (256 on a pair of CTAs) x BN columns
//   weights   dW[e] = sum of X[row(r)]^T dY[r]   tiles of 128 (256) features of X x BN features of dY, the contraction over the rows of e
//
// Persistent CTAs (or pairs, cta_group::2), one per SM, walk the tiles; how many there are every CTA finds from the offsets when it
// begins.  All operands come by TMA: rows that lie anywhere four at a time (tile::gather4), rows that follow one another and weights in
// boxes.  A step is 128 bytes of the contraction for `rows` and 64 rows for `weights`.
//
//   warps 0..3    gathered rows of X, where they are gathered
//   warp  4       boxes; announces the bytes of a stage
//   warp  5       tensor-memory allocation; four tcgen05.mma a stage, issued by the leader of a pair for both CTAs
//   warps 8..15   read-out: tensor memory -> (scales) -> rows of the output; zeros for rows that belong to no expert
//
// What bounds it: long contractions the MMAs, in a long loop of them the power limit; short ones the read-out, which shares the shared memory with
// the loads and the MMAs (65536 rows, 256 -> 1024: 43 us, 29 without read-out, 34 without its stores; stores straight from the registers, 32
// bytes a lane, 49).  16-bit, 64 experts, 2048 -> 512: 65536 rows 110 us = 1.25 PFLOP/s, 131072 rows 210 us = 1.31, weight gradients 136 and
// 240-260; 8-bit integers 60 and 105-130 us = 2.1-2.6 POP/s, 8192 rows of 4096 -> 4096 76-86 us = 3.2-3.6.
// Rows leave in the operands' 16 bits, rounded once, or in float32 where the caller asks for that: a weighted sum of 16-bit rows is then off by
// 0.0024 (relative 2-norm, bf16) where one rounding of the sum alone makes 0.0017, and a training step that has its rows in float32 takes half
// as long again (65536 rows, 1024 x 256: 202 us -> 306; 131072 of 2048 x 512: 895 -> 1235), so the caller decides.
// Brought to the L2 a tile ahead by bulk prefetches, gathered rows came later, not sooner (131072 rows: 220 -> 259 us).
//
// Experts differ in size, and a weight gradient's tile takes as long as its expert has rows.  So the contraction of a large expert is cut
// into ranges of at most `range_steps` steps, a CTA's share of all steps (half of it: more sums of ranges; 65536 rows of 64 experts, the
// largest 4858, 1024 x 256: 71 us, the whole share 54); tiles go out largest range first, every second
// round of the CTAs backwards.  Ranges of a cut expert leave float32 sums in the workspace, which a second kernel adds in the order of
// the rows: the same bits in every run.  64 experts of 100 to 5000 rows, 1024 x 256 features: tiles in the experts' order, uncut, kept the
// tensor cores of one pair busy for 61 % of 106 us and those of another for 4 %.
//
// Rows of a tile that belong to the next expert are computed and not stored.  In a contraction over rows they would do harm, even where
// the other operand is 0 (0 * infinity), so the last step of an expert takes the rows behind its end from outside the tensor: zeros.
#include <type_traits>

#include "egs_tcgen05.cuh"

namespace egs {

namespace {

constexpr int kGatherWarps = 4, kBoxWarp = 4, kIssueWarp = 5, kReadWarp0 = 8, kReadWarps = 8;
constexpr int kRaggedThreads = (kReadWarp0 + kReadWarps) * 32;
constexpr uint32_t kRaggedHeader = 512;
constexpr uint32_t kATile = 16384;                 // 128 rows x 128 bytes, or 64 rows x 128 features of 2 bytes
constexpr uint32_t kSegBytes = 8192;               // 64 rows x 128 bytes: a column segment of a tile whose rows are the contraction's
constexpr uint32_t kReadArea = 4096;               // transpose of a read-out warp
constexpr size_t kRaggedSmem = 227 * 1024;
constexpr int kSmCount = 148;

struct __align__(16) RaggedHeader {
  unsigned long long full[kMaxStages];
  unsigned long long empty[kMaxStages];
  unsigned long long acc_full[2];
  unsigned long long acc_empty[2];
  unsigned long long drain;
  uint32_t tmem_base;
  uint32_t abort_flag;
  int warp_sums[2 * kRaggedThreads / 32];
  int ranges;
};
static_assert(sizeof(RaggedHeader) <= kRaggedHeader, "header does not fit");

struct RaggedTiles {
  int BN, stages, steps;       // steps: of `rows`
  int tiles_n, tiles_c;        // column tiles; `weights`: tiles over X's features
  int range_steps;             // `weights`: steps of a range at most
  int most_ranges;             // ... and how many there can be
  float* partial;              // ... sums of the ranges of cut experts [range, C, N]
  int gathers;                 // X's rows are gathered
  int vectors;                 // rows of the output begin on 16 bytes and are whole 16 bytes
  int words;                   // ... on 4 bytes, whole 4 bytes (16-bit output): 1; on 8 and whole 8: 2
  uint32_t table_bytes;        // of each of the two tables
  Div by_n, by_c;
};

// The right operand's part of a stage: rows of 128 bytes for its columns (weights [E, N, C]), else column segments of 64.
__host__ __device__ constexpr uint32_t b_tile_bytes(int columns, bool rows) {
  return rows ? static_cast<uint32_t>(columns) * 128u : static_cast<uint32_t>((columns + 63) / 64) * kSegBytes;
}

template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
  if (PAIR) tma_load_3d_pair(dst, map, x, y, z, bar);
  else tma_load_3d(dst, map, x, y, z, bar);
}
template <bool PAIR>
__device__ __forceinline__ void load_rows4(uint32_t dst, const void* map, int x, int r0, int r1, int r2, int r3, uint32_t bar) {
  if (PAIR)
    tma_gather4_pair(dst, map, x, r0, r1, r2, r3, bar);
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
        : "memory");
}

// Four contraction steps of 32 bytes of 8-bit integers (16-bit operands: umma_f16_x4).
#define EGS_I8_X4(GROUP)                                                    \
  asm volatile(                                                             \
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"                        \
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"                   \
      "tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], %1, %2, %3, p;\n\t"  \
      "add.u64 a, %1, 2;\n\tadd.u64 b, %2, 2;\n\t"                          \
      "tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %3, q;\n\t"    \
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"                            \
      "tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %3, q;\n\t"    \
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"                            \
      "tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %3, q;\n\t}"   \
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)    \
      : "memory")
template <bool PAIR>
__device__ __forceinline__ void umma_i8_x4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if (PAIR) EGS_I8_X4("2");
  else EGS_I8_X4("1");
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

// The row ranges of a weight gradient, in shared memory.
struct Ranges {
  int* first;       // rows [first, end)
  int* end;
  int* expert;
  int* partial;     // place among the ranges of cut experts, -1 where the expert is not cut
  int* order;       // ranges by descending size
};
__host__ __device__ constexpr uint32_t range_bytes(int most) { return static_cast<uint32_t>(5 * most * 4 + 15) & ~15u; }
__device__ __forceinline__ Ranges ranges_at(unsigned char* mem, int most) {
  int* p = reinterpret_cast<int*>(mem);
  return {p, p + most, p + 2 * most, p + 3 * most, p + 4 * most};
}
constexpr int kStepRows = 64;        // contraction rows of a step of a weight gradient
__host__ __device__ inline int steps_of(int rows) { return (rows + kStepRows - 1) / kStepRows; }
// Ranges of an expert with that many rows.
__device__ __forceinline__ int ranges_of(int rows, int range_steps) {
  const int steps = steps_of(rows);
  return steps <= range_steps ? 1 : (steps + range_steps - 1) / range_steps;
}

// Exclusive sums of `a` and `b` over the threads of the CTA, and the totals; `sums`: an int a warp and quantity.
__device__ __forceinline__ void scan_two(int& a, int& b, int& total_a, int& total_b, int* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kRaggedThreads / 32;
  const int own_a = a, own_b = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int va = __shfl_up_sync(0xffffffffu, a, o), vb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += va;
      b += vb;
    }
  }
  if (lane == 31) {
    sums[warp] = a;
    sums[warps + warp] = b;
  }
  __syncthreads();
  total_a = total_b = 0;
  int before_a = 0, before_b = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) {
      before_a += sums[w];
      before_b += sums[warps + w];
    }
    total_a += sums[w];
    total_b += sums[warps + w];
  }
  a += before_a - own_a;
  b += before_b - own_b;
  __syncthreads();
}

template <typename OutT>
__device__ __forceinline__ uint32_t pack_out(uint32_t a, uint32_t b) { return pack2(static_cast<OutT*>(nullptr), a, b); }

// T: operands' type (int8_t: with scales), OutT: the output's.
template <typename T, typename OutT, bool WEIGHTS, bool PAIR>
__global__ void __cluster_dims__(PAIR ? 2 : 1, 1, 1) __launch_bounds__(kRaggedThreads, 1)
ragged_kernel(const __grid_constant__ RaggedParams p, const __grid_constant__ RaggedTiles q, const __grid_constant__ TensorMap3 map_a,
              const __grid_constant__ TensorMap3 map_a4, const __grid_constant__ TensorMap3 map_b, const __grid_constant__ TensorMap3 map_b4) {
  constexpr bool kInt8 = sizeof(T) == 1, kTwoBytes = sizeof(OutT) == 2;
  constexpr int kBlock = PAIR ? 256 : 128;           // rows of a tile
  constexpr int kStepElems = 128 / sizeof(T);        // `rows`
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  RaggedHeader* hdr = reinterpret_cast<RaggedHeader*>(smem_raw);
  int* offsets = reinterpret_cast<int*>(smem_raw + kRaggedHeader);
  int* starts = reinterpret_cast<int*>(smem_raw + kRaggedHeader + q.table_bytes);      // row blocks before each expert's
  const uint32_t smem0 = smem_u32(smem_raw);
  const Ranges range = ranges_at(smem_raw + kRaggedHeader + q.table_bytes, q.most_ranges);
  const uint32_t ring0 = (smem0 + kRaggedHeader + q.table_bytes + (WEIGHTS ? range_bytes(q.most_ranges) : q.table_bytes) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? static_cast<int>(blockIdx.x & 1) : 0;
  const bool leader = rank == 0;
  const int columns = PAIR ? q.BN / 2 : q.BN;        // of the right operand, staged by this CTA
  const uint32_t stage_bytes = kATile + b_tile_bytes(columns, !WEIGHTS && p.nc);
  const uint32_t area0 = ring0 + static_cast<uint32_t>(q.stages) * stage_bytes;
  const uint32_t acc_cols = tmem_cols_for(q.BN);
  volatile uint32_t* abort_flag = &hdr->abort_flag;
  const int first_unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, unit_stride = PAIR ? gridDim.x >> 1 : gridDim.x;

  // ---- set-up ----
  if (tid == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(smem_u32(&hdr->full[s]), 1);
      mbar_init(smem_u32(&hdr->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&hdr->acc_full[b]), 1);
      mbar_init(smem_u32(&hdr->acc_empty[b]), PAIR ? 2 * kReadWarps : kReadWarps);     // (a pair's: the leader's copy is used)
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
    for (int e = tid; e <= p.E; e += kRaggedThreads) offsets[e] = p.offsets[e];
  else if (tid < 2)
    offsets[tid] = tid ? p.rows : 0;
  __syncthreads();
  if (warp == kIssueWarp) {
    if (PAIR) {
      tmem_alloc2(smem_u32(&hdr->tmem_base), 2u * acc_cols);
      tmem_relinquish2();
    } else {
      tmem_alloc(smem_u32(&hdr->tmem_base), 2u * acc_cols);
      tmem_relinquish();
    }
  }
  {
    int carry = 0, carry_cut = 0;                    // blocks (ranges), ranges of cut experts
    for (int e0 = 0; e0 < p.E; e0 += kRaggedThreads) {
      const int e = e0 + tid, rows = e < p.E ? offsets[e + 1] - offsets[e] : 0;
      const int own = e >= p.E ? 0 : WEIGHTS ? ranges_of(rows, q.range_steps) : (rows + kBlock - 1) / kBlock;
      int at = own, cut = WEIGHTS && own > 1 ? own : 0, total, total_cut;
      scan_two(at, cut, total, total_cut, hdr->warp_sums);
      at += carry;
      cut += carry_cut;
      carry += total;
      carry_cut += total_cut;
      if constexpr (!WEIGHTS) {
        if (e < p.E) starts[e] = at;
        if (e == p.E - 1) starts[p.E] = carry;
      } else {
        const int steps = steps_of(rows), each = own ? (steps + own - 1) / own * kStepRows : 0;
        for (int i = 0; i < own; ++i) {
          range.first[at + i] = min(offsets[e] + i * each, offsets[e + 1]);
          range.end[at + i] = min(offsets[e] + (i + 1) * each, offsets[e + 1]);
          range.expert[at + i] = e;
          range.partial[at + i] = own > 1 ? cut + i : -1;
        }
        if (tid == 0) hdr->ranges = carry;
      }
    }
    if constexpr (WEIGHTS) {
      __syncthreads();
      const int n = hdr->ranges;
      for (int i = tid; i < n; i += kRaggedThreads) {
        const int size = range.end[i] - range.first[i];
        int before = 0;
        for (int j = 0; j < n; ++j) {
          const int other = range.end[j] - range.first[j];
          before += other > size || (other == size && j < i) ? 1 : 0;
        }
        range.order[before] = i;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();                      // both CTAs' barriers are initialised before anything crosses the pair
  tc_fence_after();
  const uint32_t tmem_base = hdr->tmem_base;
  const int units = WEIGHTS ? hdr->ranges * q.tiles_n * q.tiles_c : starts[p.E] * q.tiles_n;
  const uint32_t full0 = PAIR ? map_to_cta(smem_u32(&hdr->full[0]), 0) : smem_u32(&hdr->full[0]);
  // tile `round` of this CTA or pair
  auto unit_of = [&](int round) { return round * unit_stride + (WEIGHTS && (round & 1) ? unit_stride - 1 - first_unit : first_unit); };
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
      if constexpr (!WEIGHTS) {
        int e = 0;
        for (int round = 0, u; (u = unit_of(round)) < units && alive; ++round) {
          const int block = q.by_n.quotient(u);
          e = expert_of(starts, p.E, block, e);
          const int r = offsets[e] + (block - starts[e]) * kBlock + rank * 128 + warp * 32 + lane;
          const int mine = r < offsets[e + 1] ? p.by_k.quotient(p.slots[r]) : -1;
          int row[8][4];
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) row[i][j] = __shfl_sync(0xffffffffu, mine, i * 4 + j);
          for (int ks = 0; ks < q.steps; ++ks) {
            if (!wait_free()) break;
            const uint32_t bar = full0 + at.slot * 8u;
            const uint32_t dst = ring0 + static_cast<uint32_t>(at.slot) * stage_bytes + static_cast<uint32_t>(warp) * 4096u;
            at.next(q.stages);
            if (elect_one()) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                load_rows4<PAIR>(dst + i * 512u, &map_a4, ks * kStepElems, row[i][0], row[i][1], row[i][2], row[i][3], bar);
            }
          }
        }
      } else {
        // a warp has 16 rows of every step; lanes 16..31 look up those of the step behind
        for (int round = 0, u; (u = unit_of(round)) < units && alive; ++round) {
          int x = q.by_n.quotient(u);
          const int c = q.by_c.remainder(x), i = range.order[x];
          const int begin = range.first[i], end = range.end[i];
          auto look = [&](int step) {                // (an even one)
            const int r = begin + (step + (lane >> 4)) * kStepRows + warp * 16 + (lane & 15);
            return r < end ? p.slots[r] : -1;
          };
          const int steps = steps_of(end - begin);
          const int f0 = c * kBlock + rank * 128;
          int coming = steps ? look(0) : -1, now = -1;
          for (int ks = 0; ks < steps; ++ks) {
            if (!(ks & 1)) {
              now = coming < 0 ? -1 : p.by_k.quotient(coming);
              coming = ks + 2 < steps ? look(ks + 2) : -1;
            }
            int row[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) row[i][j] = __shfl_sync(0xffffffffu, now, (ks & 1) * 16 + i * 4 + j);
            if (!wait_free()) break;
            const uint32_t bar = full0 + at.slot * 8u;
            const uint32_t dst = ring0 + static_cast<uint32_t>(at.slot) * stage_bytes + static_cast<uint32_t>(warp) * 2048u;
            at.next(q.stages);
            if (elect_one()) {
#pragma unroll
              for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  load_rows4<PAIR>(dst + s * kSegBytes + i * 512u, &map_a4, f0 + s * 64, row[i][0], row[i][1], row[i][2], row[i][3], bar);
            }
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
      int steps = q.steps, a0 = 0, f0 = 0, begin = 0, end = 0;
      if constexpr (!WEIGHTS) {
        e = expert_of(starts, p.E, x, e);
        a0 = offsets[e] + (x - starts[e]) * kBlock + rank * 128;
      } else {
        int y = x;
        f0 = q.by_c.remainder(y) * kBlock + rank * 128;
        y = range.order[y];
        begin = range.first[y];
        end = range.end[y];
        steps = steps_of(end - begin);
      }
      for (int ks = 0; ks < steps; ++ks) {
        if (!wait_free()) break;
        const uint32_t own = smem_u32(&hdr->full[at.slot]), bar = full0 + at.slot * 8u;
        const uint32_t a_dst = ring0 + static_cast<uint32_t>(at.slot) * stage_bytes, b_dst = a_dst + kATile;
        at.next(q.stages);
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(own, bytes);
          if constexpr (!WEIGHTS) {
            if (!q.gathers) load_box<PAIR>(a_dst, &map_a, ks * kStepElems, a0, 0, bar);
            if (p.nc) {
              load_box<PAIR>(b_dst, &map_b, ks * kStepElems, n0, e, bar);
            } else {
              for (int s = 0; s * 64 < columns; ++s) load_box<PAIR>(b_dst + s * kSegBytes, &map_b, n0 + s * 64, ks * kStepElems, e, bar);
            }
          } else {
            const int r0 = begin + ks * kStepRows;
            if (r0 + kStepRows <= end) {
              if (!q.gathers)
                for (int s = 0; s < 2; ++s) load_box<PAIR>(a_dst + s * kSegBytes, &map_a, f0 + s * 64, r0, 0, bar);
              for (int s = 0; s * 64 < columns; ++s) load_box<PAIR>(b_dst + s * kSegBytes, &map_b, n0 + s * 64, r0, 0, bar);
            } else {                                 // the last rows of the expert, zeros behind them
              for (int i = 0; i < kStepRows / 4; ++i) {
                const int r = r0 + i * 4;
                const int ra = r < end ? r : -1, rb = r + 1 < end ? r + 1 : -1, rc = r + 2 < end ? r + 2 : -1, rd = r + 3 < end ? r + 3 : -1;
                if (!q.gathers)
                  for (int s = 0; s < 2; ++s) load_rows4<PAIR>(a_dst + s * kSegBytes + i * 512u, &map_a4, f0 + s * 64, ra, rb, rc, rd, bar);
                for (int s = 0; s * 64 < columns; ++s)
                  load_rows4<PAIR>(b_dst + s * kSegBytes + i * 512u, &map_b4, n0 + s * 64, ra, rb, rc, rd, bar);
              }
            }
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == kIssueWarp) {
    // =========================== MMA issuer ===========================
    if (leader) {
      const bool b_mn = WEIGHTS || !p.nc;
      const uint64_t a_desc = WEIGHTS ? make_smem_desc(0u, kSegBytes, 1024u) : make_smem_desc(0u, 16u, 1024u);
      const uint64_t b_desc = (b_mn ? make_smem_desc(0u, kSegBytes, 1024u) : make_smem_desc(0u, 16u, 1024u)) + (kATile >> 4);
      const uint32_t a_adv = (WEIGHTS ? 16u * 128u : 32u) >> 4, b_adv = (b_mn ? 16u * 128u : 32u) >> 4;
      // 8-bit integers: signed operands (format 1), int32 accumulator (format 2 in the place of 1)
      const uint32_t idesc = kInt8 ? make_idesc(1u, 0u, 0u, kBlock, q.BN) + (1u << 4)
                                   : make_idesc(sizeof(T) == 2 ? Elem<typename std::conditional<kInt8, __half, T>::type>::fmt : 0u, WEIGHTS ? 1u : 0u,
                                                b_mn ? 1u : 0u, kBlock, q.BN);
      int t = 0;                                     // tiles with an accumulator
      for (int round = 0, u; (u = unit_of(round)) < units && alive; ++round) {
        int steps = q.steps;
        if constexpr (WEIGHTS) {
          int x = q.by_n.quotient(u);
          x = range.order[q.by_c.quotient(x)];
          steps = steps_of(range.end[x] - range.first[x]);
          if (steps == 0) continue;
        }
        const int buf = t & 1;
        if (t >= 2) {
          alive = mbar_wait_all<PAIR>(smem_u32(&hdr->acc_empty[buf]), ((t >> 1) - 1) & 1, abort_flag, p.status.word);
          if (!alive) break;
        }
        ++t;
        const uint32_t d = tmem_base + static_cast<uint32_t>(buf) * acc_cols;
        for (int ks = 0; ks < steps; ++ks) {
          alive = mbar_wait_all<PAIR>(smem_u32(&hdr->full[at.slot]), at.round & 1, abort_flag, p.status.word);
          if (!alive) break;
          const uint32_t empty = smem_u32(&hdr->empty[at.slot]);
          const uint32_t addr = (ring0 + static_cast<uint32_t>(at.slot) * stage_bytes) >> 4;
          at.next(q.stages);
          tc_fence_after();
          if (elect_one()) {
            if constexpr (kInt8) umma_i8_x4<PAIR>(d, a_desc + addr, b_desc + addr, idesc, ks > 0 ? 1u : 0u);
            else umma_f16_x4<PAIR>(d, a_desc + addr, b_desc + addr, a_adv, b_adv, idesc, ks > 0 ? 1u : 0u);
            umma_done<PAIR>(empty);
            if (ks + 1 == steps) umma_done<PAIR>(smem_u32(&hdr->acc_full[buf]));
          }
        }
      }
    }
    pdl_trigger();
    __syncwarp();
  } else if (warp >= kReadWarp0) {
    // =========================== read-out ===========================
    const int ew = warp - kReadWarp0, lg = ew & 3, share = ew >> 2;     // TMEM lane group (warp number mod 4), share of the column blocks
    const uint32_t area = area0 + static_cast<uint32_t>(ew) * kReadArea;
    const uint32_t lane_base = static_cast<uint32_t>(lg * 32) << 16;
    OutT* out = static_cast<OutT*>(p.Out);
    if (!WEIGHTS && p.offsets) {                     // rows that belong to no expert
      const long long begin = static_cast<long long>(offsets[p.E]) * p.N, end = static_cast<long long>(p.rows) * p.N;
      const long long step = static_cast<long long>(gridDim.x) * (kReadWarps * 32);
      for (long long i = begin + blockIdx.x * (kReadWarps * 32) + ew * 32 + lane; i < end; i += step) out[i] = from_f32<OutT>(0.f);
    }
    // What is known about a tile before its accumulator is there, asked for while the tile before is read out: the two loads that find a
    // row's scale took a microsecond of every tile.
    struct Tile {
      int e, n0, bn, rows, partial;      // rows: of the warp's 32 that are stored
      long long row0;                    // output row of the first of them
      bool have;                         // there is an accumulator (an expert without rows: zeros)
      float scale, w_scale[4];           // 8-bit operands: of this lane's row, of its columns (32 apart)
    };
    int e_last = 0;
    auto tile_of = [&](int u) {
      Tile x{};
      const int block = q.by_n.quotient(u);
      x.n0 = (u - block * q.tiles_n) * q.BN;
      x.bn = min(q.BN, p.N - x.n0);
      x.partial = -1;
      if constexpr (!WEIGHTS) {
        x.e = e_last = expert_of(starts, p.E, block, e_last);
        const int r = offsets[x.e] + (block - starts[x.e]) * kBlock + rank * 128 + lg * 32;
        x.row0 = r;
        x.rows = min(32, offsets[x.e + 1] - r);
        x.have = true;
        if constexpr (kInt8) {
          if (lane < x.rows) x.scale = p.a_scale[p.slots ? p.by_k.quotient(p.slots[r + lane]) : r + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = kTwoBytes ? (i >> 1) * 128 + share * 64 + (i & 1) * 32 : i * 64 + share * 32;
            if (c + lane < x.bn) x.w_scale[i] = p.w_scale[static_cast<long long>(x.e) * p.N + x.n0 + c + lane];
          }
        }
      } else {
        int y = block;
        const int f = q.by_c.remainder(y) * kBlock + rank * 128 + lg * 32;
        y = range.order[y];
        x.partial = range.partial[y];
        x.row0 = static_cast<long long>(x.partial >= 0 ? x.partial : range.expert[y]) * p.C + f;
        x.rows = min(32, p.C - f);
        x.have = range.end[y] > range.first[y];
      }
      return x;
    };
    int t = 0;
    Tile tile{}, coming{};
    if (unit_of(0) < units) coming = tile_of(unit_of(0));
    for (int round = 0; unit_of(round) < units && alive; ++round) {
      tile = coming;
      if (unit_of(round + 1) < units) coming = tile_of(unit_of(round + 1));
      const int n0 = tile.n0, bn = tile.bn, rows = tile.rows, partial = tile.partial;
      const long long row0 = tile.row0;
      const bool have = tile.have;
      const int buf = t & 1;
      if (have) {
        alive = mbar_wait_all(smem_u32(&hdr->acc_full[buf]), (t >> 1) & 1, abort_flag, p.status.word);
        if (!alive) break;
        ++t;
        tc_fence_after();
      }
      const uint32_t acc = tmem_base + lane_base + static_cast<uint32_t>(buf) * acc_cols;
      bool released = false;
      auto release = [&]() {
        if (!have || released) return;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&hdr->acc_empty[buf]), 0));
          else mbar_arrive(smem_u32(&hdr->acc_empty[buf]));
        }
        released = true;
      };
      // 32 columns of the accumulator in float32
      auto read = [&](int c, int which, uint32_t (&v)[32]) {
        if (have) {
          tmem_ld32(acc + static_cast<uint32_t>(c), v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        if constexpr (kInt8) {                       // (which: the block's place among those of the warp)
          const uint32_t scales = area0 + kReadWarps * kReadArea + static_cast<uint32_t>(ew) * 128u;
          const float own = which == 0 ? tile.w_scale[0] : which == 1 ? tile.w_scale[1] : which == 2 ? tile.w_scale[2] : tile.w_scale[3];
          __syncwarp();
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + lane * 4u), "f"(own) : "memory");
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float w[4];
            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]) : "r"(scales + i * 4u) : "memory");
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i + k] = __float_as_uint(static_cast<float>(static_cast<int>(v[i + k])) * (tile.scale * w[k]));
          }
        }
      };
      auto store_f32 = [&](float* to, bool vectors) {
        for (int c = share * 32; c < bn; c += 64) {
          uint32_t v[32];
          read(c, c >> 6, v);
          if (c + 64 >= bn) release();
          warp_regs_emit(v, area, lane, [&](int row, int cj, uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
            const int col = c + cj;
            if (row >= rows || col >= bn) return;
            float* o = to + (row0 + row) * p.N + n0 + col;
            if (vectors) {
              store4(o, x0, x1, x2, x3);
            } else {
              o[0] = __uint_as_float(x0);
              if (col + 1 < bn) o[1] = __uint_as_float(x1);
              if (col + 2 < bn) o[2] = __uint_as_float(x2);
              if (col + 3 < bn) o[3] = __uint_as_float(x3);
            }
          });
        }
      };
      if (WEIGHTS && partial >= 0) {
        store_f32(q.partial, p.N % 4 == 0);
      } else if constexpr (sizeof(OutT) == 2) {
        // 64 columns = 128 bytes of a row at a time, eight lanes to a row
        for (int c = share * 64; c < bn; c += 128) {
          const uint32_t srow = area + static_cast<uint32_t>(lane) * 128u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (c + h * 32 < bn) {
              uint32_t v[32];
              read(c + h * 32, (c >> 7) * 2 + h, v);
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
          } else if (q.words == 2) {                 // rows of whole double words: two at a time
            const int col = c + (lane & 15) * 4;
#pragma unroll
            for (int it = 0; it < 16; ++it) {
              const int row = it * 2 + (lane >> 4);
              uint2 y;
              asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(y.x), "=r"(y.y) : "r"(area + row * 128u + (static_cast<uint32_t>(((lane & 15) >> 1) ^ (row & 7)) << 4) + (lane & 1) * 8u) : "memory");
              if (row < rows && col < bn) *reinterpret_cast<uint2*>(out + (row0 + row) * p.N + n0 + col) = y;
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
        store_f32(reinterpret_cast<float*>(out), q.vectors);
      }
      release();                                     // (warps whose share of the columns is empty)
    }
  }

  // ---- common exit (see dense16_kernel) ----
  tc_fence_before();
  __syncthreads();
  if (!PAIR) {
    if (warp == kIssueWarp) tmem_release(tmem_base, 2u * acc_cols, smem_u32(&hdr->drain), abort_flag, p.status, lane);
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
      tmem_dealloc2(tmem_base, 2u * acc_cols);
    }
  }
}

// dW of cut experts: the sums of their ranges, in order.  fours: every expert's begins on four elements and is a whole number of them.
template <typename T>
__global__ void __launch_bounds__(256) ragged_join_kernel(const int* offsets, const float* partial, T* out, long long size, int E, int range_steps, bool fours) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  long long base = 0;
  int turn = 0;                                // every gridDim.y-th cut expert is this CTA's
  for (int e0 = 0; e0 < E; e0 += 32) {         // a lane looks at an expert
    const int own = e0 + lane < E ? ranges_of(offsets[e0 + lane + 1] - offsets[e0 + lane], range_steps) : 1;
    for (unsigned cut = __ballot_sync(0xffffffffu, own > 1); cut; cut &= cut - 1) {
      const int n = __shfl_sync(0xffffffffu, own, __ffs(cut) - 1);
      const float* p = partial + base * size;
      base += n;
      if (turn++ % gridDim.y != blockIdx.y) continue;
      T* o = out + (e0 + __ffs(cut) - 1) * size;
      if (fours) {
        for (long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 4; i < size; i += static_cast<long long>(gridDim.x) * 1024) {
          float4 sum = *reinterpret_cast<const float4*>(p + i);
#pragma unroll 4
          for (int r = 1; r < n; ++r) {
            const float4 x = *reinterpret_cast<const float4*>(p + r * size + i);
            sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
          }
          store4(o + i, __float_as_uint(sum.x), __float_as_uint(sum.y), __float_as_uint(sum.z), __float_as_uint(sum.w));
        }
      } else {
        for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < size; i += static_cast<long long>(gridDim.x) * 256) {
          float sum = p[i];
#pragma unroll 4
          for (int r = 1; r < n; ++r) sum += p[r * size + i];
          o[i] = from_f32<T>(sum);
        }
      }
    }
  }
}

template <typename T, typename OutT, bool WEIGHTS, bool PAIR>
cudaError_t launch_ragged(const RaggedParams& p, RaggedTiles q, long long most_units, const TensorMap3 (&maps)[4], cudaStream_t st) {
  q.table_bytes = static_cast<uint32_t>((p.E + 1) * 4 + 15) & ~15u;
  const size_t before = (kRaggedHeader + q.table_bytes + (WEIGHTS ? range_bytes(q.most_ranges) : q.table_bytes) + 1023u) & ~static_cast<size_t>(1023);
  const size_t stage = kATile + b_tile_bytes(PAIR ? q.BN / 2 : q.BN, !WEIGHTS && p.nc);
  const size_t fixed = before + kReadWarps * (kReadArea + (sizeof(T) == 1 ? 128 : 0));
  q.stages = static_cast<int>((kRaggedSmem - fixed) / stage);
  if (q.stages > kMaxStages) q.stages = kMaxStages;
  cudaError_t err = ensure_smem_optin<ragged_kernel<T, OutT, WEIGHTS, PAIR>>(static_cast<int>(kRaggedSmem));
  if (err != cudaSuccess) return err;
  const long long workers = PAIR ? kSmCount / 2 : kSmCount;
  const long long grid = (most_units < workers ? (most_units < 1 ? 1 : most_units) : workers) * (PAIR ? 2 : 1);
  count_launch();
  return launch_kernel(ragged_kernel<T, OutT, WEIGHTS, PAIR>, static_cast<unsigned>(grid), kRaggedThreads, fixed + q.stages * stage, st, true, p, q,
                       maps[0], maps[1], maps[2], maps[3]);
}

// Maps of a matrix [rows, width] with a pitch: boxes of `box_rows` rows of 128 bytes, and four rows one by one.
bool row_maps(TensorMap3* box, TensorMap3* four, const void* base, int elem, long long rows, int width, long long pitch, int box_rows) {
  const unsigned long long dims[3] = {static_cast<unsigned long long>(width), static_cast<unsigned long long>(rows), 1ull};
  const unsigned long long strides[2] = {static_cast<unsigned long long>(pitch) * elem, static_cast<unsigned long long>(pitch) * elem * rows};
  const unsigned b3[3] = {static_cast<unsigned>(128 / elem), static_cast<unsigned>(box_rows), 1u}, b2[2] = {static_cast<unsigned>(128 / elem), 1u};
  return encode_tensor_map_strided(box, base, elem, 3, dims, strides, b3) && encode_tensor_map_strided(four, base, elem, 2, dims, strides, b2);
}

template <typename T, typename OutT, bool WEIGHTS>
cudaError_t launch_by_pair(const RaggedParams& p, const RaggedTiles& q, bool pair, long long units, const TensorMap3 (&maps)[4], cudaStream_t st) {
  return pair ? launch_ragged<T, OutT, WEIGHTS, true>(p, q, units, maps, st) : launch_ragged<T, OutT, WEIGHTS, false>(p, q, units, maps, st);
}

// The tile that takes the least time by this estimate, in clocks.  A step of a CTA costs its bytes at 60 a clock (what the L2 gives all SMs) or its
// MMAs where they take longer (two clocks a column in both types: 8-bit steps have twice the elements, at twice the rate); a read-out, under the
// next tile's steps all but the last, `fixed` and 3000 or 4500 for 256 columns.  blocks(rows of a tile): tiles of one column.  The widest tile on
// pairs or single CTAs moves the fewest bytes; another has to be a tenth faster.
struct TileChoice {
  bool pair;
  int BN;
};
template <class Blocks>
TileChoice choose_tile(int N, long long steps, int elem, bool pairs, Blocks&& blocks) {
  constexpr TileChoice kCandidates[] = {{true, 256}, {false, 256}, {true, 128}, {false, 128}, {false, 64}};
  const double fixed = elem == 1 ? 2500 : 1500, wide = elem == 1 ? 4500 : 3000;
  TileChoice best{false, 64};
  double least = -1;
  for (const TileChoice& c : kCandidates) {
    if ((c.BN > 64 && N <= c.BN / 2) || (c.pair && !pairs)) continue;
    const int workers = c.pair ? kSmCount / 2 : kSmCount;
    const double bytes = kATile + b_tile_bytes(c.pair ? c.BN / 2 : c.BN, false), mma = 2 * c.BN;
    const double work = (bytes / 60 > mma ? bytes / 60 : mma) * steps, out = fixed + wide * c.BN / 256;
    const long long units = static_cast<long long>(blocks(c.pair ? 256 : 128) * ((N + c.BN - 1) / c.BN));
    const double time = static_cast<double>((units + workers - 1) / workers) * (work > out ? work : out) + out;
    if (least < 0 || time < (best.BN == 256 && c.BN < 256 ? 0.9 : 1.0) * least) {
      least = time;
      best = c;
    }
  }
  return best;
}

int words_of(const RaggedParams& p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.Out);
  return p.N % 4 == 0 && (at & 7u) == 0 ? 2 : p.N % 2 == 0 && (at & 3u) == 0 ? 1 : 0;
}

// Tiles of one width, no wider than they need be: 776 columns are four of 224, not of 256.  (tcgen05.mma: multiples of 16, of 32 for a pair.)
int even_width(int N, int BN) {
  const int tiles = (N + BN - 1) / BN;
  return ((N + tiles - 1) / tiles + 31) / 32 * 32;
}

}  // namespace

cudaError_t launch_ragged_rows_tensor(const RaggedParams& p, int dtype, int out_dtype, cudaStream_t st) {
  const int elem = dtype == EGS_I8 ? 1 : 2;
  const int out_elem = out_dtype == EGS_F32 ? 4 : 2;
  RaggedTiles q{};
  q.steps = (p.C * elem + 127) / 128;
  // (an expert's last block is half empty in the mean)
  const int experts = p.offsets ? (p.rows < p.E ? p.rows : p.E) : 1;
  const double each = static_cast<double>(p.rows) / experts;
  const TileChoice tile = choose_tile(p.N, q.steps, elem, true, [&](int rows) { return experts * (each <= rows / 2 ? 1.0 : !p.offsets ? (p.rows + rows - 1) / rows : each / rows + 0.5); });
  const bool pair = tile.pair;
  q.BN = even_width(p.N, tile.BN);
  const int block = pair ? 256 : 128;
  q.tiles_n = (p.N + q.BN - 1) / q.BN;
  q.by_n = Div(q.tiles_n);
  q.gathers = p.slots != nullptr;
  q.vectors = (static_cast<long long>(p.N) * out_elem) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.Out) & 15u) == 0;
  q.words = words_of(p);
  const long long blocks = p.offsets ? p.rows / block + (p.rows < p.E ? p.rows : p.E) : (p.rows + block - 1) / block;
  const int columns = pair ? q.BN / 2 : q.BN;
  TensorMap3 maps[4];
  if (!row_maps(&maps[0], &maps[1], p.A, elem, p.a_rows, p.C, p.a_row, 128)) return cudaErrorInvalidValue;
  const unsigned long long dims[3] = {static_cast<unsigned long long>(p.nc ? p.C : p.N), static_cast<unsigned long long>(p.nc ? p.N : p.C),
                                      static_cast<unsigned long long>(p.E)};
  const unsigned long long strides[2] = {static_cast<unsigned long long>(p.w_row) * elem, static_cast<unsigned long long>(p.w_expert) * elem};
  const unsigned box[3] = {static_cast<unsigned>(128 / elem), p.nc ? static_cast<unsigned>(columns) : 64u, 1u};
  if (!encode_tensor_map_strided(&maps[2], p.W, elem, 3, dims, strides, box)) return cudaErrorInvalidValue;
  maps[3] = maps[2];
  const long long units = blocks * q.tiles_n;
  if (dtype == EGS_I8) {
    if (out_dtype == EGS_F16) return launch_by_pair<int8_t, __half, false>(p, q, pair, units, maps, st);
    if (out_dtype == EGS_BF16) return launch_by_pair<int8_t, __nv_bfloat16, false>(p, q, pair, units, maps, st);
    return launch_by_pair<int8_t, float, false>(p, q, pair, units, maps, st);
  }
  const bool wide = out_dtype == EGS_F32;
  if (dtype == EGS_F16)
    return wide ? launch_by_pair<__half, float, false>(p, q, pair, units, maps, st) : launch_by_pair<__half, __half, false>(p, q, pair, units, maps, st);
  return wide ? launch_by_pair<__nv_bfloat16, float, false>(p, q, pair, units, maps, st)
              : launch_by_pair<__nv_bfloat16, __nv_bfloat16, false>(p, q, pair, units, maps, st);
}

// (a range below this takes less time than the kernel that joins ranges)
constexpr int kLeastRange = 24;

// How a weight gradient is cut: see the top of the file.  Ranges of cut experts have more than half of range_steps steps each.
struct DweightPlan {
  bool pair;
  RaggedTiles q;
  long long most_partial;
};
static DweightPlan dweight_plan(const RaggedParams& p) {
  DweightPlan d{};
  RaggedTiles& q = d.q;
  // where experts are cut, tiles of any size fill the SMs
  const int each = steps_of(p.rows) / p.E + 1;
  const bool pairs = p.C > 128 && p.rows >= 256ll * p.E;
  const TileChoice tile = each > kLeastRange ? TileChoice{pairs && p.N > 64, p.N > 128 ? 256 : p.N > 64 ? 128 : 64}
                                             : choose_tile(p.N, each, 2, pairs, [&](int features) { return static_cast<double>((p.C + features - 1) / features) * p.E; });
  d.pair = tile.pair;
  const int block = d.pair ? 256 : 128, workers = d.pair ? kSmCount / 2 : kSmCount;
  q.BN = even_width(p.N, tile.BN);
  q.tiles_n = (p.N + q.BN - 1) / q.BN;
  q.tiles_c = (p.C + block - 1) / block;
  const long long steps = steps_of(p.rows), share = steps * q.tiles_n * q.tiles_c / workers;
  q.range_steps = static_cast<int>(share < kLeastRange ? kLeastRange : share < steps ? share : steps);
  if (each > q.range_steps) {
    // the mean expert is cut: into as many ranges as leave the last round of the CTAs fullest (one of 1024 steps and 20 tiles: 8 ranges are 2.2
    // rounds, 7 are 1.9), each range costing what its sums take to be written and read
    const double sums = 8.0 * p.E * p.C * p.N / 2.9e6;           // steps of 0.45 us at 6.5 TB/s
    double least = -1;
    for (int n = 1; n <= 16; ++n) {
      const long long units = static_cast<long long>(p.E) * n * q.tiles_n * q.tiles_c;
      const int steps_each = (each + n - 1) / n;
      if (steps_each < kLeastRange) break;
      const double time = static_cast<double>((units + workers - 1) / workers) * steps_each + (n > 1 ? n * sums : 0.0);
      if (least < 0 || time < least) {
        least = time;
        q.range_steps = steps_each;
      }
    }
  }
  d.most_partial = steps <= q.range_steps ? 0 : 2 * (steps / q.range_steps) + 2;
  q.most_ranges = static_cast<int>(p.E + d.most_partial);
  return d;
}
size_t ragged_dweight_workspace(const RaggedParams& p) { return static_cast<size_t>(dweight_plan(p).most_partial) * p.C * p.N * sizeof(float); }

cudaError_t launch_ragged_dweight_tensor(const RaggedParams& p, int dtype, void* workspace, cudaStream_t st) {
  DweightPlan d = dweight_plan(p);
  RaggedTiles& q = d.q;
  q.by_n = Div(q.tiles_n);
  q.by_c = Div(q.tiles_c);
  q.partial = static_cast<float*>(workspace);
  q.gathers = p.slots != nullptr;
  q.vectors = (p.N * 2ll) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.Out) & 15u) == 0;
  q.words = words_of(p);
  TensorMap3 maps[4];
  if (!row_maps(&maps[0], &maps[1], p.A, 2, p.a_rows, p.C, p.a_row, 64) || !row_maps(&maps[2], &maps[3], p.W, 2, p.rows, p.N, p.w_row, 64))
    return cudaErrorInvalidValue;
  const long long units = static_cast<long long>(q.most_ranges) * q.tiles_c * q.tiles_n, size = static_cast<long long>(p.C) * p.N;
  cudaError_t err = dtype == EGS_F16 ? launch_by_pair<__half, __half, true>(p, q, d.pair, units, maps, st)
                                     : launch_by_pair<__nv_bfloat16, __nv_bfloat16, true>(p, q, d.pair, units, maps, st);
  if (err != cudaSuccess || d.most_partial == 0) return err;
  // (six CTAs an SM at most: most experts are not cut, and 16 rows of CTAs that find nothing to add took 2 to 6 us more)
  const dim3 ctas(static_cast<unsigned>(size / 1024 < 1 ? 1 : size / 1024 > kSmCount ? kSmCount : size / 1024), p.E < 6 ? p.E : 6);
  const bool fours = size % 4 == 0 && (reinterpret_cast<uintptr_t>(p.Out) & 7u) == 0;
  count_launch();
  if (dtype == EGS_F16)
    return launch_kernel(ragged_join_kernel<__half>, ctas, 256, 0, st, true, p.offsets, q.partial, static_cast<__half*>(p.Out), size, p.E, q.range_steps, fours);
  return launch_kernel(ragged_join_kernel<__nv_bfloat16>, ctas, 256, 0, st, true, p.offsets, q.partial, static_cast<__nv_bfloat16*>(p.Out), size, p.E,
                       q.range_steps, fours);
}

}  // namespace egs
