// Attention of a ragged batch of new tokens over a paged key/value history
// (sm_100a): the kernel for many query rows per key head, on the 5th
// generation tensor cores.
//
// The query rows of one key head (tokens x query heads of the group) are
// packed into blocks of 256: two tiles of 128, the M of tcgen05.mma and the
// lanes of tensor memory.  A CTA (one per SM, persistent; its run of tiles
// from paged.cuh) works on one block at a time, 128 keys a step:
//   warp 10    walks the run and hands out its pieces; loads K of a step and V of
//              the step before into a ring of tiles, one TMA box per page
//              (128-byte swizzle);
//   warps 8, 9 issue S = Q K^T and O += P V for a tile each (d = 128: warp 8
//              for both), P taken from
//              tensor memory;
//   warp 11    brings in a piece's queries (cp.async; d = 128: of tile 0, warp 9
//              of tile 1), and overwrites rows of V that must not count, at the
//              edges;
//   warps 0-3  and 4-7: the softmax of tile 0 and of tile 1, one row a
//              thread: scores from tensor memory, mask at the edges, running
//              maximum, exponentials, and the weights back into tensor memory
//              (bf16, over the scores' columns).
// While one tile's weights are formed the tensor cores work for the other.
// The reference that the weights are taken against moves only when a score
// exceeds it by more than 8 in base 2 (d = 128: when a step's weights add up
// to more than 2^16): until then weights grow, which float32 sums hold as well,
// and the output rows in tensor memory need no rescaling; when it does, the
// row's own thread rescales them.
//
// What bounds it: a step of 256 rows x 128 keys is 32768 exponentials, 2048
// clocks of an SM's 16 a clock, against 1024 (d = 64) or 2048 (d = 128) clocks
// of tensor-core time.  2048 tokens over 14,300 positions, 20 heads: d = 64
// 232 us, 693 TF/s, about 2800 clocks a step: a tile's exponentials 1400 (1024 at
// the full rate, one warp a scheduler at a time), its loads, maximum, stores and
// barriers as long, behind the other tile's exponentials; d = 128 309 us, 1040
// TF/s, about 3950 clocks a step, the chain of one tile's weights (2300) and the
// two products after them (1060, and 600 between the issue of one and the sight
// of the other's end).
//
// Rounding: scores, maxima, sums and outputs are float32; the weights enter
// the second product as bf16, the operand type of the tensor cores (half a
// step is 2^-8 of each weight; the sums take the unrounded ones), and the
// result is rounded once.
//
// Keys and values outside what a block reads: pages wholly outside are not
// loaded, and on the block's first and last tile the rows of V outside are
// overwritten with zeros in shared memory, as a weight of zero does not
// silence an infinity there; scores outside are replaced, not added to.
//
// Tensor-core operations of one thread run in the order of their issue: the
// next scores overwrite a tile's weights right behind the product that reads
// them.  Every mbarrier wait is bounded (~2 s, MOSS_ERR_TIMEOUT).
#include <math_constants.h>

#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace moss {
namespace pattn {
namespace {

constexpr int kTileRows = 128;
constexpr int kThreads = 384;
constexpr int kMmaWarp = 8;   // and 9: one for each tile of rows
constexpr int kLoadWarp = 10, kEdgeWarp = 11;
// Registers a thread: launched with 168 (65536 / 384, the multiple of 8 below),
// then moved from the third warpgroup to the two that hold 128 scores a
// thread: 2 * 216 + 72 = 3 * 168.  (2048 tokens over 14k positions, d = 64 / 128:
// 216 250 / 316 us; 208 263 / 329; with 224 the others spill; both before the
// turns' barriers were preceded by a __syncwarp, 238 since.)
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * 168,
              "setmaxnreg draws on the launch's registers");
constexpr int kKeys = kTcTile;  // keys per step
constexpr uint32_t kSub = kKeys * 128;  // 128 rows x 64 columns of bf16
constexpr uint32_t kTmemCols = 512;

constexpr float kSlack = 8.0f;
// d = 128: the sum of a tile's weights above which the reference is raised by a power
// of two before the next tile, and the sum above which the tile is done again by its
// true maximum.  Between the two a tile's products are formed with weights that
// large, so the second leaves float32 sums room for values up to 2^55.
constexpr float kRaiseAbove = 0x1p16f, kRedoAbove = 0x1p64f;
// Tiles that would run in step (each finds its next scores ready, d = 64) and
// leave the special-function unit idle between the exponentials take turns
// instead: one's loads and stores lie behind the other's exponentials.
template <int D>
constexpr bool kTurns = D == 64;
struct TcArgs {
  CUtensorMap k_map;  // pages as [pages * hkv * page_size, d], box {64, min(page_size, 128)}
  CUtensorMap v_map;
  Args a;
};

// Tensor memory has room for scores (2 x 128 columns), outputs (2 x d) and
// weights (2 x 64) at d = 64: the next step's scores are then formed while the
// softmax works on this step's, as soon as it holds them in registers.
template <int D>
constexpr bool kOwnP = 2 * kKeys + 2 * D + kKeys <= static_cast<int>(kTmemCols);
// The ring holds tiles of K and V in the order in which they are used: step n's
// K and step n - 1's V.  At d = 64 the two share a barrier (one wait less a
// step); at d = 128 five tiles fit, each with its own.
template <int D>
constexpr int kSlots = D == 64 ? 12 : 5;
template <int D>
constexpr bool kPaired = D == 64;
template <int D>
constexpr int kIssuers = D == 64 ? 2 : 1;  // threads that issue the products
static_assert(kOwnP<64> && !kOwnP<128>, "the order of issue below");

// Shared memory after the 1024-byte alignment: queries of both tiles, the
// ring, the mbarriers.
template <int D>
constexpr uint32_t kTileBytes = kSub * (D / 64);

// One piece of work, as the load warp (which walks the run) hands it to the
// others; steps == 0 ends them.
struct Job {
  int steps, tile;        // steps, and the first one's tile of the sequence
  int lo, hi;             // keys that the block reads
  int row0, rr0, h, rows; // the sequence's first packed row; the block's first row, head, rows
  int pos0;               // position of the sequence's first new token
  int whole, slot;        // all of the item, or the slot of a cut piece
  int from[2], to[2];     // steps that each tile of rows takes part in
};
constexpr int kJobs = 3;
constexpr int kJobReaders = 8 + 2 + 1;  // softmax warps, warps 8 and 9, the edge warp
struct Bars {
  unsigned long long full[6], empty[6];  // a slot, or a pair of slots
  unsigned long long q_full[2], s_full[2], s_free[2], p_full[2], pv_done[2], done[2];
  unsigned long long job_full[kJobs], job_empty[kJobs], q_free[2];
  unsigned long long edge_in, edge;  // V of an edge tile has landed; is ready
  int64_t scan[kThreads / 32];
  Run run;
  uint32_t tmem;
  int gave_up;  // a wait ran out: the others stop waiting too
  Job jobs[kJobs];
};
template <int D>
constexpr size_t tc_smem() {
  return 1024 + kTileBytes<D> * (2 + kSlots<D>) + sizeof(Bars);
}

// K-major operand (Q, K): 128-byte rows, 128-byte swizzle, 8-row groups 1024
// bytes apart.
__device__ __forceinline__ uint64_t k_major(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}
// MN-major operand (V as [keys][d]): 64 values of d per 128-byte row, 8-key
// groups 1024 bytes apart, the next 64 values of d one sub-tile further.
__device__ __forceinline__ uint64_t mn_major(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFF) |
         (static_cast<uint64_t>(kSub >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16, D float32, A and B bf16, M = 128; bit 16: B is MN-major.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTileRows >> 4) << 24);
}
// One thread of a converged warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
// 32 consecutive columns of this thread's TMEM lane, no wait.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Waits for this thread's TMEM loads; the registers go through so that no use
// of them moves above the wait.
__device__ __forceinline__ void tmem_ld_wait(uint32_t* r) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
        "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]),
        "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// Bits n and up of 32.
__device__ __forceinline__ uint32_t bits_from(int n) {
  return n <= 0 ? 0xffffffffu : (n >= 32 ? 0u : 0xffffffffu << n);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Waits on the critical path poll without suspending (the wake-up costs more
// than a step can hide).  Bounded as everywhere: the first to run out records
// the timeout and makes every later wait of the CTA return at once, so that all
// roles run to their end on whatever the buffers hold (addresses never depend
// on data) and the kernel returns.
__device__ __forceinline__ bool test_phase(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// SUSPEND: the instruction that may suspend the thread for a while, for waits
// off the critical path, whose polling would take issue slots from the softmax.
constexpr uint32_t kWaitLimit = static_cast<uint32_t>(kWaitLimitNs >> 20);
template <bool SUSPEND>
__device__ __forceinline__ void wait_phase(unsigned long long* bar, uint32_t parity,
                                           volatile int* gave_up, uint32_t limit = kWaitLimit) {
  const uint32_t at = pipe::smem_u32(bar);
  parity &= 1;
  uint32_t start = 0;
#pragma unroll 1
  for (uint32_t n = 1; !(SUSPEND ? pipe::mbar_try_wait(bar, parity) : test_phase(at, parity));
       ++n) {
    if (SUSPEND || (n & 1023) == 0) {
      const uint32_t now = static_cast<uint32_t>(global_ns() >> 20);  // about a millisecond
      if (start == 0) start = now;
      if (*gave_up) return;
      if (now - start > limit) {
        *gave_up = 1;
        record_device_error(MOSS_ERR_TIMEOUT);
        return;
      }
    }
  }
}
// A pair of float32 in one 64-bit register: one instruction for both.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split_pair(uint64_t x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The two tiles' turns at the exponentials: barrier 1 + w is passed by tile w's
// threads once the other tile's have arrived.
__device__ __forceinline__ void turn_wait(int w) {
  // the instruction wants the warp together; and nothing of the exponentials
  // moves ahead of it then (250 us without, 238 with)
  __syncwarp();
  asm volatile("barrier.sync.aligned %0, %1;" ::"r"(1 + w), "n"(2 * kTileRows) : "memory");
}
__device__ __forceinline__ void turn_pass(int w) {
  __syncwarp();
  asm volatile("barrier.arrive.aligned %0, %1;" ::"r"(1 + w), "n"(2 * kTileRows) : "memory");
}

// Whether `x` holds for all threads of both tiles (barrier 3).
__device__ __forceinline__ bool all_of_both(bool x) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.red.and.pred q, 3, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(x)), "n"(2 * kTileRows)
      : "memory");
  return all != 0;
}

// Steps [from, to) of the piece that tile w of its rows takes part in.
__device__ __forceinline__ void tile_span(const Args& a, const paged::Seq& seq,
                                          const paged::Piece& p, const paged::Range& r, int w,
                                          int& from, int& to) {
  from = to = 0;
  const int r0 = p.block * kTcRows + w * kTileRows;
  const int rest = paged::rows_of(a.split, seq) - r0;
  if (rest <= 0) return;
  const int last_row = r0 + (rest < kTileRows ? rest : kTileRows) - 1;
  const int pos0 = seq.len - seq.t;
  const int lo = paged::window_start(pos0 + paged::quotient(r0, a.split.group), a.split.context);
  const int hi = pos0 + paged::quotient(last_row, a.split.group) + 1;
  if (hi <= lo) return;
  const int base = r.tile0 + p.tile;
  from = lo / kKeys - base;
  to = (hi - 1) / kKeys + 1 - base;
  if (from < 0) from = 0;
  if (to > p.n) to = p.n;
  if (from >= to) from = to = 0;
}

// Step j of the piece has keys that its block does not read.
__device__ __forceinline__ bool is_edge(const Job& job, int j) {
  const int key0 = (job.tile + j) * kKeys;
  return key0 < job.lo || key0 + kKeys > job.hi;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    tc_kernel(const __grid_constant__ TcArgs args) {
  extern __shared__ unsigned char smem_raw[];
  const Args& a = args.a;
  unsigned char* sb =
      smem_raw + ((1024u - (pipe::smem_u32(smem_raw) & 1023u)) & 1023u);
  constexpr uint32_t kBytes = kTileBytes<D>;
  constexpr int kRing = kPaired<D> ? kSlots<D> / 2 : kSlots<D>;  // barriers
  constexpr uint32_t kSpan = kPaired<D> ? 2 * kBytes : kBytes;   // bytes of each
  unsigned char* q_smem = sb;                  // two tiles
  unsigned char* ring = sb + 2 * kBytes;
  Bars& bars = *reinterpret_cast<Bars*>(ring + kRing * kSpan);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x, ctas = gridDim.x;

  if (tid == 0) {
    prefetch_map(&args.k_map);
    prefetch_map(&args.v_map);
    for (int i = 0; i < kRing; ++i) {
      pipe::mbar_init(&bars.full[i], 1);
      pipe::mbar_init(&bars.empty[i], kIssuers<D>);
    }
    for (int w = 0; w < 2; ++w) {
      pipe::mbar_init(&bars.q_full[w], 1);
      pipe::mbar_init(&bars.q_free[w], 1);
      pipe::mbar_init(&bars.s_full[w], 1);
      pipe::mbar_init(&bars.s_free[w], kTileRows);
      pipe::mbar_init(&bars.p_full[w], kTileRows);
      pipe::mbar_init(&bars.pv_done[w], 1);
      pipe::mbar_init(&bars.done[w], 1);
    }
    pipe::mbar_init(&bars.edge_in, kIssuers<D>);
    for (int i = 0; i < kJobs; ++i) {
      pipe::mbar_init(&bars.job_full[i], 1);
      pipe::mbar_init(&bars.job_empty[i], kJobReaders);
    }
    pipe::mbar_init(&bars.edge, 1);
    bars.gave_up = 0;
    pipe::fence_mbar_init();
  }
  if (warp == kMmaWarp) tc::alloc(&bars.tmem, kTmemCols);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  // longer batches than a warp looks through need the whole CTA
  if (a.batch.s > kWarpSeqs) find_runs<kThreads, 1>(a, cta, ctas, bars.scan, &bars.run);
  const uint32_t tmem = bars.tmem;
  // Tensor memory: scores of both tiles, outputs of both tiles, then the weights
  // in columns of their own where there is room (d = 64), else over the scores
  // that they come from.

  // Reads the jobs in order: the next one, and the end of its use.
  uint32_t job_turn = 0;
  auto next_job = [&]() -> const Job& {
    wait_phase<true>(&bars.job_full[job_turn % kJobs], job_turn / kJobs, &bars.gave_up);
    return bars.jobs[job_turn % kJobs];
  };
  // After a wait that ran out a job may never come: its steps count as none (the
  // same for the whole warp).
  auto alive = [&](const Job& job) {
    return __all_sync(0xffffffffu,
                      job.steps > 0 && *static_cast<volatile int*>(&bars.gave_up) == 0) != 0;
  };

  // Brings the queries of tile w of a piece into the K-major, swizzled operand, as
  // soon as the piece before has formed its last scores (whole warp; `made`: of
  // the pieces before).
  auto load_queries = [&](const Job& job, int w, uint32_t& made) {
    if (job.from[w] >= job.to[w]) return;
    if (made > 0) {
      if (lane == 0) wait_phase<true>(&bars.q_free[w], made - 1, &bars.gave_up);
      __syncwarp();
    }
    ++made;
    // kStep rows at a time, a row's 16-byte chunks side by side; the row's token
    // and head of the group advance without a division
    constexpr int kChunks = D / 8, kStep = 32 / kChunks;
    const int group = static_cast<int>(a.split.group.d);
    const int c = lane % kChunks, row0 = lane / kChunks;
    uint32_t dst = pipe::smem_u32(q_smem) + w * kBytes + (c / 8) * kSub + row0 * 128;
    const int rows = job.rows - w * kTileRows;
    const int rr = job.rr0 + w * kTileRows + row0;
    const int token = paged::quotient(rr, a.split.group);
    int head = rr - token * group;
    const int step_t = paged::quotient(kStep, a.split.group), step_h = kStep - step_t * group;
    const int64_t token_size = static_cast<int64_t>(a.hq) * D;
    const int64_t step_size = step_t * token_size + step_h * D, wrap_size = token_size - group * D;
    const uint16_t* src =
        a.q + (job.row0 + token) * token_size + (job.h * group + head) * D + c * 8;
#pragma unroll 2
    for (int r8 = 0; r8 < kTileRows; r8 += 8, dst += 1024) {
#pragma unroll
      for (int k = 0; k < 8; k += kStep) {
        // rows that do not exist are zeros
        const int n = r8 + k + row0 < rows ? 16 : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         dst + k * 128 + (((c & 7) ^ (k + row0)) << 4)),
                     "l"(n ? src : a.q), "r"(n)
                     : "memory");
        head += step_h;
        src += step_size;
        if (head >= group) {
          head -= group;
          src += wrap_size;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    tc::fence_async_shared();
    __syncwarp();
    if (lane == 0) pipe::mbar_arrive(&bars.q_full[w]);
  };

  // every warp of a warpgroup takes the same setmaxnreg
  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == kLoadWarp) {
    // ------------------------------------------------------------ loads
    // Step n, counted over all pieces, brings V of step n - 1 and its own K.
    const int box = a.batch.page_shift < 7 ? 1 << a.batch.page_shift : kKeys;
    const int boxes = kKeys / box;
    uint32_t turn = 0;      // barriers of the ring used so far
    bool any = false, ok = true;
    int v_y = -1;           // this lane's box of V for the next step (-1: none)
    uint32_t v_bytes = 0;
    auto claim = [&](uint32_t bytes) {
      const uint32_t slot = turn % kRing;
      if (lane == 0) wait_phase<true>(&bars.empty[slot], (turn / kRing) + 1, &bars.gave_up);
      __syncwarp();
      ok = __all_sync(0xffffffffu, *static_cast<volatile int*>(&bars.gave_up) == 0);
      if (ok) {
        if (lane == 0) pipe::mbar_arrive_expect_tx(&bars.full[slot], bytes);
        ++turn;
      }
      __syncwarp();
      return slot;
    };
    auto fetch = [&](const CUtensorMap* map, uint32_t slot, uint32_t offset, int y) {
      if (!ok || y < 0) return;
      const uint32_t dst = pipe::smem_u32(ring + slot * kSpan) + offset + lane * box * 128;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) tma_load(dst + c * kSub, map, c * 64, y, &bars.full[slot]);
    };
    auto load = [&](int k_y, uint32_t k_bytes) {
      if constexpr (kPaired<D>) {
        const uint32_t slot = claim(v_bytes + k_bytes);
        fetch(&args.v_map, slot, 0, v_y);
        fetch(&args.k_map, slot, kBytes, k_y);
      } else {
        fetch(&args.v_map, claim(v_bytes), 0, v_y);
        if (ok) fetch(&args.k_map, claim(k_bytes), 0, k_y);
      }
      any = true;
      v_y = k_y;
      v_bytes = k_bytes;
    };
    Run run;
    if (a.batch.s <= kWarpSeqs) {
      run = warp_run(a, cta, ctas, [&](int s) { return seq_work(a, s); });
    } else {
      run = bars.run;
    }
    if (lane == 0) clear_note(a, cta);
    paged::Walker walk;
    paged::Piece p{};
    paged::Range range{};
    if (run.count > 0) walk.start(a.batch, a.split, run.s, run.offset, run.count);
    walk.left = run.count;
    uint32_t made = 0;
    auto hand_out = [&](int steps) {
      const uint32_t slot = made % kJobs;
      if (lane == 0) {
        wait_phase<true>(&bars.job_empty[slot], made / kJobs + 1, &bars.gave_up);
        // a reader may still be at the slot if the wait ran out: nothing but zeros
        // is written over its job then
        if (*static_cast<volatile int*>(&bars.gave_up) != 0) steps = 0;
        Job job{};
        job.steps = steps;
        if (steps > 0) {
          job.tile = range.tile0 + p.tile;
          job.lo = range.lo;
          job.hi = range.hi;
          job.row0 = walk.seq.row0;
          job.rr0 = p.block * kTcRows;
          job.h = p.h;
          const int rest = paged::rows_of(a.split, walk.seq) - job.rr0;
          job.rows = rest < kTcRows ? rest : kTcRows;
          job.pos0 = walk.seq.len - walk.seq.t;
          job.whole = p.whole;
          job.slot = p.whole ? 0 : slot_of(p, cta);
          tile_span(a, walk.seq, p, range, 0, job.from[0], job.to[0]);
          tile_span(a, walk.seq, p, range, 1, job.from[1], job.to[1]);
          if (!p.whole) note_piece(a, p, range, walk.seq, run, cta);
          check_length(a, p.s, walk.seq);
        }
        bars.jobs[slot] = job;
        pipe::mbar_arrive(&bars.job_full[slot]);
      }
      ++made;
      __syncwarp();
    };
    while (ok && walk.next(a.batch, a.split, p, range)) {
      hand_out(p.n);
      const int32_t* table = a.batch.table + static_cast<int64_t>(p.s) * a.batch.max_pages;
      const int base = range.tile0 + p.tile;
      auto page_of = [&](int j) {
        const int at = (base + j) * kKeys + lane * box;
        if (lane >= boxes || j >= p.n || at >= range.hi || at + box <= range.lo) return -2;
        return table[at >> a.batch.page_shift];
      };
      int next = page_of(0);
      for (int j = 0; j < p.n && ok; ++j) {
        int page = next;
        next = page_of(j + 1);
        if (page != -2 && (page < 0 || page >= a.batch.pages)) {
          record_device_error(MOSS_ERR_VALUE);
          page = -2;
        }
        const int at = (base + j) * kKeys + lane * box;
        load(page == -2 ? -1
                        : ((page * a.split.hkv + p.h) << a.batch.page_shift) +
                              (at & ((1 << a.batch.page_shift) - 1)),
             static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, page != -2))) *
                 static_cast<uint32_t>(box) * 128u * (D / 64));
      }
    }
    if (ok && any) load(-1, 0);  // the last V
    hand_out(0);
    // copies still in flight land before this CTA may retire
    if (!ok) {
      for (uint32_t i = turn > kRing ? turn - kRing : 0; i < turn; ++i)
        pipe::mbar_wait(&bars.full[i % kRing], (i / kRing) & 1);
    }
    __syncwarp();
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // ------------------------------------------------------------ products
    // Per step S, and O += P V of the step before.  d = 64: a warp for each tile
    // of rows.  d = 128: one for both, as the order of the products is what
    // keeps the two tiles' softmaxes out of step there.  The warp stays together
    // and one elected thread issues: issued from a branch of one lane, a product of
    // 64 clocks took 75 to 110 to issue, and the issue bounded the kernel.
    if (warp - kMmaWarp < kIssuers<D>) {
      constexpr int kEach = 2 / kIssuers<D>;
      const int w0 = warp - kMmaWarp;
      uint32_t turn = 0;  // barriers of the ring passed
      uint32_t edges = 0;
      uint32_t q_seen[kEach] = {}, p_seen[kEach] = {}, s_made[kEach] = {};  // phases passed
      bool v_on[kEach] = {}, v_first[kEach] = {}, v_edge = false;  // the step whose V comes next
      int from[kEach] = {}, to[kEach] = {};
      const uint32_t ring_u = pipe::smem_u32(ring), q_u = pipe::smem_u32(q_smem);
      auto wait = [&](unsigned long long* bar, uint32_t parity) {
        wait_phase<false>(bar, parity, &bars.gave_up);
        __syncwarp();
        tc::fence_after();
      };
      auto tile_at = [&](uint32_t n) { return ring_u + n % kRing * kSpan; };
      auto edge = [&] {
        if (!v_edge) return;
        if (elect_one()) pipe::mbar_arrive(&bars.edge_in);
        wait(&bars.edge, edges++);
      };
      auto release = [&](uint32_t slot) {
        if (elect_one()) tc::commit(&bars.empty[slot]);
        __syncwarp();
      };
      auto product = [&](int x, uint32_t v) {
        if (!v_on[x]) return;
        const int w = w0 + x;
        wait(&bars.p_full[w], p_seen[x]++);
        const uint32_t o = tmem + 2 * kKeys + w * D;
        const uint32_t weights =
            kOwnP<D> ? tmem + 2 * kKeys + 2 * D + w * (kKeys / 2) : tmem + w * kKeys;
        const uint64_t values = mn_major(v);
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i)
            mma_ts(o, weights + i * 8, values + i * (2048 >> 4), idesc(D, true),
                   (!v_first[x] || i > 0) ? 1u : 0u);
          tc::commit(&bars.pv_done[w]);
        }
        __syncwarp();
      };
      auto scores = [&](int x, int j, uint32_t k) {
        if (j < from[x] || j >= to[x]) return;
        const int w = w0 + x;
        if (j == from[x]) wait(&bars.q_full[w], q_seen[x]++);
        // the softmax holds the tile's previous scores in registers
        if (kOwnP<D> && s_made[x] > 0) wait(&bars.s_free[w], s_made[x] - 1);
        ++s_made[x];
        const uint64_t queries = k_major(q_u + w * kBytes), keys = k_major(k);
        const bool last = j + 1 == to[x];
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const uint32_t off = ((i / 4) * kSub + (i % 4) * 32) >> 4;
            mma_ss(tmem + w * kKeys, queries + off, keys + off, idesc(kKeys, false), i > 0);
          }
          tc::commit(&bars.s_full[w]);
          if (last) tc::commit(&bars.q_free[w]);
        }
        __syncwarp();
      };
      for (;;) {
        const Job& job = next_job();
        if (!alive(job)) break;
        const int steps = job.steps, lo = job.lo, hi = job.hi, key_tile = job.tile;
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
          from[x] = job.from[w0 + x];
          to[x] = job.to[w0 + x];
        }
        __syncwarp();
        if (lane == 0) pipe::mbar_arrive(&bars.job_empty[job_turn % kJobs]);
        ++job_turn;
#pragma unroll 1
        for (int j = 0; j < steps; ++j) {
          const uint32_t slot = turn % kRing, tile = tile_at(turn);
          wait(&bars.full[slot], turn / kRing);
          if constexpr (kPaired<D>) {
            // Where the weights have columns of their own the scores need not
            // wait for them; but a piece's first queries wait for the piece
            // before.
            if (j > 0) scores(0, j, tile + kBytes);
            edge();
            product(0, tile);
            if (j == 0) scores(0, j, tile + kBytes);
            release(slot);
            ++turn;
          } else {
            // (a piece's first queries wait for both products of the piece before;
            // the keys are waited for here, off the path from weights to scores)
            const uint32_t k_slot = (turn + 1) % kRing, k = tile_at(turn + 1);
            wait(&bars.full[k_slot], (turn + 1) / kRing);
            edge();
            product(0, tile);
            if (j == 0) product(kEach - 1, tile);
            scores(0, j, k);
            if (j > 0) product(kEach - 1, tile);
            release(slot);
            scores(kEach - 1, j, k);
            release(k_slot);
            turn += 2;
          }
#pragma unroll
          for (int x = 0; x < kEach; ++x) {
            v_on[x] = j >= from[x] && j < to[x];
            v_first[x] = j == from[x];
          }
          const int key0 = (key_tile + j) * kKeys;
          v_edge = key0 < lo || key0 + kKeys > hi;
        }
      }
      if (turn > 0) {
        wait(&bars.full[turn % kRing], turn / kRing);
        edge();
#pragma unroll
        for (int x = 0; x < kEach; ++x) product(x, tile_at(turn));
      }
    }
    // d = 128: the warp without products brings in the queries of tile 1.
    if (warp - kMmaWarp >= kIssuers<D>) {
      uint32_t q_made = 0;
      for (;;) {
        const Job& job = next_job();
        if (!alive(job)) break;
        load_queries(job, 1, q_made);
        if (lane == 0) pipe::mbar_arrive(&bars.job_empty[job_turn % kJobs]);
        ++job_turn;
      }
    }
    // every product and every commit has landed before tensor memory and
    // this CTA's shared memory are given back
    __syncwarp();
    unsigned long long* done = &bars.done[warp - kMmaWarp];
    if (elect_one()) tc::commit(done);
    __syncwarp();
    pipe::mbar_wait(done, 0);
    __syncwarp();
  } else if (warp == kEdgeWarp) {
    // ------------------------------------------------------------ queries, edges
    // Per piece: the queries (d = 128: of tile 0), then rows of V that no row of the
    // block attends to.
    uint32_t turn = 0, edges = 0, q_made[2] = {0, 0};
    for (;;) {
      const Job& job = next_job();
      if (!alive(job)) break;
#pragma unroll 1
      for (int w = 0; w < kIssuers<D>; ++w) load_queries(job, w, q_made[w]);
      for (int j = 0; j < job.steps; ++j) {
        turn += kPaired<D> ? 1 : 2;  // V of this step comes with the next
        if (!is_edge(job, j)) continue;
        if (lane == 0) wait_phase<true>(&bars.edge_in, edges, &bars.gave_up);
        ++edges;
        __syncwarp();
        unsigned char* v = ring + turn % kRing * kSpan;
        const int key0 = (job.tile + j) * kKeys;
        // a row's chunks side by side; rows before `lo`, then rows from `hi`
        const int before = job.lo - key0 < 0 ? 0 : (job.lo - key0 < kKeys ? job.lo - key0 : kKeys);
        const int after = job.hi - key0 < 0 ? 0 : (job.hi - key0 < kKeys ? job.hi - key0 : kKeys);
        constexpr int kChunks = D / 8;
        const int c = lane % kChunks;
        unsigned char* column = v + (c / 8) * kSub + (c % 8) * 16;
        const int r0 = lane / kChunks;
#pragma unroll 4
        for (int r = r0; r < before; r += 32 / kChunks)
          *reinterpret_cast<uint4*>(column + r * 128) = make_uint4(0, 0, 0, 0);
#pragma unroll 4
        for (int r = after + r0; r < kKeys; r += 32 / kChunks)
          *reinterpret_cast<uint4*>(column + r * 128) = make_uint4(0, 0, 0, 0);
        tc::fence_async_shared();
        __syncwarp();
        if (lane == 0) pipe::mbar_arrive(&bars.edge);
      }
      if (lane == 0) pipe::mbar_arrive(&bars.job_empty[job_turn % kJobs]);
      ++job_turn;
    }
  }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int w = warp >> 2;
    const int r = tid & (kTileRows - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + w * kKeys + lanes;
    const uint32_t o_at = tmem + 2 * kKeys + w * D + lanes;
    const uint32_t p_at =
        (kOwnP<D> ? tmem + 2 * kKeys + 2 * D + w * (kKeys / 2) : tmem + w * kKeys) + lanes;
    uint32_t seen = 0;  // score tiles taken so far
    auto wait = [&](unsigned long long* bar, uint32_t parity) {
      wait_phase<false>(bar, parity, &bars.gave_up);
      __syncwarp();
      tc::fence_after();
    };
    const int group = static_cast<int>(a.split.group.d);
    for (;;) {
      const Job& job = next_job();
      __syncwarp();
      const int steps = job.steps, from = job.from[w], to = job.to[w], key_tile = job.tile;
      const int rows = job.rows - w * kTileRows;  // of this tile, if positive
      const bool whole = job.whole;
      const int64_t slot = job.slot;
      const bool turns = kTurns<D> && job.rows > kTileRows;
      // this row's place in q and out, and its position; rows that do not exist
      // follow the last one (their queries are zeros)
      const int rr0 = job.rr0 + w * kTileRows;
      const bool row_on = r < rows;
      const int rr = rr0 + (row_on ? r : (rows > 0 ? rows - 1 : 0));
      const int t = paged::quotient(rr, a.split.group);
      const int pos = job.pos0 + t;
      const int64_t row_at =
          ((static_cast<int64_t>(job.row0) + t) * a.hq + job.h * group + (rr - t * group)) * D;
      // keys that every row of the tile attends to
      const int free_to = job.pos0 + paged::quotient(rr0, a.split.group);
      const int free_from = paged::window_start(
          job.pos0 + paged::quotient(rr0 + (rows < kTileRows ? rows : kTileRows) - 1, a.split.group),
          a.split.context);
      // Where the tiles take turns, which no limit bounds, all eight warps go on
      // with a job or none does: a wait that runs out may be seen by some only.
      // (The job is read before it is asked whether one did.)
      asm volatile("" ::: "memory");
      if (!(kTurns<D> ? all_of_both(alive(job)) : alive(job))) break;
      if (lane == 0) pipe::mbar_arrive(&bars.job_empty[job_turn % kJobs]);
      ++job_turn;
      if (rows <= 0) continue;
      if (turns && w == 1) turn_pass(0);
      float m = -CUDART_INF_F, l = 0.0f;  // reference (base 2, scaled) and sum
      float raise = 0.0f;
      if (turns || from < to) {
#pragma unroll 1
        for (int j = turns ? 0 : from; j < (turns ? steps : to); ++j) {
          if (j < from || j >= to) {
            turn_wait(w);
            if (w == 0 || j + 1 < steps) turn_pass(w ^ 1);
            continue;
          }
          wait(&bars.s_full[w], seen);
          uint32_t s[kKeys];
          const int key0 = (key_tile + j) * kKeys;
          const bool edge = key0 + kKeys - 1 > free_to || key0 < free_from;
          auto load_scores = [&] {
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld32(s_at + i * 32, s + i * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld_wait(s + i * 32);
            if (edge) {
              // keys [low, high] of the tile are this row's
              const int low = paged::window_start(pos, a.split.context) - key0;
              const int high = pos - key0;
#pragma unroll
              for (int g = 0; g < kKeys; g += 32) {
                const uint32_t on = bits_from(low - g) & ~bits_from(high + 1 - g);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(on & (1u << i))) s[g + i] = __float_as_uint(-CUDART_INF_F);
              }
            }
          };
          load_scores();
          if (kOwnP<D>) {
            tc::fence_before();
            pipe::mbar_arrive(&bars.s_free[w]);
          }
          // The reference that the weights are taken against (m, base 2, scaled).
          // d = 64: the running maximum, moved when a score exceeds it by more
          // than 8.  d = 128, where the softmax lies between two products: the
          // row's maximum over its first tile with a key, raised by whole powers of
          // two when a tile's weights add up to more than 2^16, so that most tiles
          // need no maximum.
          auto rescale = [&](float f) {
            wait(&bars.pv_done[w], seen - 1);
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
              uint32_t o[32];
              tmem_ld32(o_at + i, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(o_at + i, o);
            }
            // a step may rescale twice (raised, then far above the reference all the
            // same): the second loads follow these stores only where they have landed
            tmem_st_wait();
            l *= f;
          };
          auto maximum = [&] {
            float t4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
            for (int i = 0; i < kKeys; i += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                t4[e] = max3(t4[e], __uint_as_float(s[i + 2 * e]),
                             __uint_as_float(s[i + 2 * e + 1]));
            return fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * a.scale2;
          };
          // raises the reference to at least `top`, the row's sums with it
          auto raise_to = [&](float top) {
            const float now = fmaxf(m, top);
            const float f = now == -CUDART_INF_F ? 1.0f : exp2_fast(m - now);
            m = now;
            if (j > from) rescale(f);
          };
          if (kOwnP<D>) {
            const float top = maximum();
            // -inf against -inf is NaN: no move
            if (j == from)
              m = top;
            else if (__any_sync(0xffffffffu, top - m > kSlack))
              raise_to(top);
          } else if (__any_sync(0xffffffffu, m == -CUDART_INF_F)) {
            // rows without a key so far hold zeros: nothing to rescale
            const float top = maximum();
            if (m == -CUDART_INF_F) m = top;
          } else if (__any_sync(0xffffffffu, raise > 0.0f)) {
            rescale(exp2_fast(-raise));
            m += raise;
          }
          const uint64_t scale = pair_of(a.scale2, a.scale2);
          float sum;
          // The weights, packed over the scores' registers.
          auto weights = [&] {
            const float shift = m == -CUDART_INF_F ? 0.0f : m;
            const uint64_t base = pair_of(-shift, -shift);
            uint64_t part[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < kKeys; i += 2) {
              float e0, e1;
              const uint64_t x =
                  fma2(pair_of(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale, base);
              split_pair(x, e0, e1);
              e0 = exp2_fast(e0);
              e1 = exp2_fast(e1);
              part[i / 2 % 2] = add2(part[i / 2 % 2], pair_of(e0, e1));
              s[i / 2] = pack_bf16x2(e0, e1);
            }
            float x, y;
            split_pair(add2(part[0], part[1]), x, y);
            sum = x + y;
          };
          if (turns) turn_wait(w);
          weights();
          if (turns && (w == 0 || j + 1 < steps)) turn_pass(w ^ 1);
          if (!kOwnP<D>) {
            if (__any_sync(0xffffffffu, !(sum < kRedoAbove))) {
              // scores far above the reference (or not finite): take the true
              // maximum and do the tile again (its scores are still there)
              load_scores();
              raise_to(maximum());
              weights();
            }
            const int exponent = static_cast<int>(__float_as_uint(sum) >> 23) - 127;
            raise = sum > kRaiseAbove ? static_cast<float>(exponent) : 0.0f;
          } else if (j > from) {
            // the product before has read the weights that these replace
            wait(&bars.pv_done[w], seen - 1);
          }
          __syncwarp();
          tmem_st32(p_at, s);
          tmem_st32(p_at + 32, s + 32);
          l += sum;
          tmem_st_wait();
          tc::fence_before();
          pipe::mbar_arrive(&bars.p_full[w]);
          ++seen;
        }
        if (from < to) wait(&bars.pv_done[w], seen - 1);
      }
      // ---- this row's result
      const bool any = from < to;
      const float inv = inverse_of(l);
      if (!whole && row_on) a.stats[slot * kTcRows + w * kTileRows + r] = make_float2(m, l);
      // cut pieces: [d / 4][rows] of four values, so that a warp's rows lie side
      // by side
      float4* part = reinterpret_cast<float4*>(a.partial) + slot * (kTcRows * (D / 4)) +
                     w * kTileRows + r;
      // (rolled, 32 columns at a time: code that runs once a piece is fetched cold,
      // and more columns spill registers)
#pragma unroll 1
      for (int i = 0; i < D; i += 32) {
        uint32_t o[32];
        __syncwarp();
        if (any) {
          tmem_ld32(o_at + i, o);
          tmem_ld_wait(o);
        }
        if (row_on) {
          if (whole) {
            uint4* dst = reinterpret_cast<uint4*>(a.out + row_at + i);
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              float f[8];
#pragma unroll
              for (int x = 0; x < 8; ++x)
                f[x] = normed(__uint_as_float(o[e + x]), inv);
              dst[e / 8] = pack_bf16x8(f);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              part[(i + e) / 4 * kTcRows] =
                  any ? make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]),
                                    __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]))
                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
        }
      }
      tc::fence_before();
    }
  }
  __syncthreads();
  tc::fence_after();
  if (warp == kMmaWarp) tc::dealloc(tmem, kTmemCols);
}

// Joins the pieces of cut items, in CTA order: block x what CTA x began, block y
// 16 columns, a thread a row.
constexpr int kJoinBatch = 2;

template <int D>
__global__ void __launch_bounds__(kTcRows) join_kernel(const __grid_constant__ Args a, int ctas) {
  cudaGridDependencySynchronize();
  const int first = blockIdx.x, row = threadIdx.x;
  const Note n = a.notes[first];
  if (n.state == 0 || n.last < first || n.last >= ctas || row >= n.rows) return;
  float v[16] = {};
  float top = -CUDART_INF_F, l = 0.0f;
  for (int k0 = first; k0 <= n.last; k0 += kJoinBatch) {
    float2 st[kJoinBatch];
    float4 x[kJoinBatch][4];
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      const int k = k0 + i;
      st[i] = make_float2(-CUDART_INF_F, 0.0f);
#pragma unroll
      for (int c = 0; c < 4; ++c) x[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (k <= n.last) {
        const int64_t slot = 2 * k + (k == first ? 1 : 0);
        st[i] = a.stats[slot * kTcRows + row];
        const float4* src = reinterpret_cast<const float4*>(a.partial) +
                            (slot * (D / 4) + blockIdx.y * 4) * kTcRows + row;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[i][c] = src[c * kTcRows];
      }
    }
    float now = top;
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) now = fmaxf(now, st[i].x);
    const float shift = now == -CUDART_INF_F ? 0.0f : now;
    const float keep = exp2_fast(top - shift);
    top = now;
    l *= keep;
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] *= keep;
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      const float g = exp2_fast(st[i].x - shift);
      l = fmaf(st[i].y, g, l);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[4 * c] = fmaf(x[i][c].x, g, v[4 * c]);
        v[4 * c + 1] = fmaf(x[i][c].y, g, v[4 * c + 1]);
        v[4 * c + 2] = fmaf(x[i][c].z, g, v[4 * c + 2]);
        v[4 * c + 3] = fmaf(x[i][c].w, g, v[4 * c + 3]);
      }
    }
  }
  const float inv = inverse_of(l);
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = normed(v[e], inv);
  const int rr = n.block * kTcRows + row;
  const int t = paged::quotient(rr, a.split.group);
  const int group = static_cast<int>(a.split.group.d);
  uint4* dst = reinterpret_cast<uint4*>(
      a.out + ((static_cast<int64_t>(n.row0) + t) * a.hq + n.h * group + (rr - t * group)) * D +
      blockIdx.y * 16);
  dst[0] = pack_bf16x8(v);
  dst[1] = pack_bf16x8(v + 8);
}

// Two warps in two waits each, one polling and one suspending, on phases that are
// completed beforehand (arrive) or never: the first wait to run out ends the others.
__global__ void wait_probe_kernel(uint32_t limit, int arrive) {
  __shared__ unsigned long long bars[2];
  __shared__ int gave_up;
  if (threadIdx.x == 0) {
    pipe::mbar_init(&bars[0], 1);
    pipe::mbar_init(&bars[1], 1);
    gave_up = 0;
    pipe::fence_mbar_init();
  }
  __syncthreads();
  if (arrive && threadIdx.x == 0) {
    pipe::mbar_arrive(&bars[0]);
    pipe::mbar_arrive(&bars[1]);
  }
  for (int i = 0; i < 2; ++i) {
    if (threadIdx.x < 32)
      wait_phase<false>(&bars[i], 0, &gave_up, limit);
    else
      wait_phase<true>(&bars[i], 0, &gave_up, limit);
  }
}

template <int D>
int launch(const Args& a, int ctas, cudaStream_t stream, const char* name) {
  TcArgs args{};
  args.a = a;
  const int page = 1 << a.batch.page_shift;
  const int box = page < kKeys ? page : kKeys;
  if (!encode_pages(&args.k_map, a.k_pages, a, D, box) ||
      !encode_pages(&args.v_map, a.v_pages, a, D, box))
    return fail(MOSS_ERR_CUDA, "%s: tensor map encoding failed", name);
  static bool configured[kMaxDevices] = {};
  allow_dynamic_smem(tc_kernel<D>, tc_smem<D>(), configured);
  const int status = launch_early(tc_kernel<D>, dim3(static_cast<unsigned>(ctas), 1, 1), kThreads,
                                  tc_smem<D>(), stream, name, args);
  if (status != MOSS_OK) return status;
  return launch_early(join_kernel<D>, dim3(static_cast<unsigned>(ctas), D / 16, 1), kTcRows, 0,
                      stream, name, a, ctas);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

}  // namespace

bool encode_pages(CUtensorMap* map, const void* pages, const Args& a, int d, int box) {
  EncodeTiled fn = encoder();
  if (!fn) return false;
  const cuuint64_t rows = (static_cast<cuuint64_t>(a.batch.pages) * a.split.hkv)
                          << a.batch.page_shift;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(d), rows};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(d) * 2};
  const cuuint32_t size[2] = {64, static_cast<cuuint32_t>(box)};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(pages), dims, strides,
            size, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

cudaError_t tc_error_word(void** word) { return cudaGetSymbolAddress(word, g_device_error); }

int launch_tc(const Args& a, int64_t d, int ctas, cudaStream_t stream, const char* name) {
  return d == 64 ? launch<64>(a, ctas, stream, name) : launch<128>(a, ctas, stream, name);
}

}  // namespace pattn
}  // namespace moss

extern "C" int moss_test_paged_wait(int64_t limit_ns, int arrive, void* stream) {
  const char* name = "moss_test_paged_wait";
  if (limit_ns < 1000 || limit_ns > 100000000)
    return moss::fail(MOSS_ERR_VALUE, "%s: limit must be 1 us to 100 ms", name);
  moss::pattn::wait_probe_kernel<<<1, 64, 0, moss::as_stream(stream)>>>(
      static_cast<uint32_t>(limit_ns >> 20), arrive ? 1 : 0);
  return moss::launch_status(name);
}
