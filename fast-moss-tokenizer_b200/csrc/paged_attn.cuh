// What the paged attention kernels share: their arguments, the search for a
// CTA's run of tiles, and the partial results of items cut between CTAs.
#pragma once

#include <cuda.h>

#include "paged.cuh"
#include "pipeline.cuh"

namespace moss {
namespace pattn {

// A worker's two cut pieces leave their rows here (see paged::share_of): slot
// 2 c holds the piece with which worker c continues an item, slot 2 c + 1 the
// piece with which it begins one; note c says what it began.
struct __align__(16) Note {
  int state;   // 0: nothing cut begins here
  int last;    // the worker with the item's last piece
  int h;       // key head
  int row0;    // the sequence's first packed row
  int block;   // row block
  int rows;    // its rows
  int pad[2];
};

struct Args {
  const uint16_t* q;        // [n, hq, d]
  const uint16_t* k_pages;  // [pages, hkv, page_size, d]
  const uint16_t* v_pages;
  uint16_t* out;            // [n, hq, d]
  Note* notes;              // [workers]
  float2* stats;            // [2 * workers][rows] running maximum (base 2, scaled) and sum
  float* partial;           // [2 * workers][rows][d] unnormalised sums
  paged::Batch batch;
  paged::Split split;
  int hq;
  int least;                // tiles a worker takes at least
  float scale2;             // scale * log2(e)
};

// Kernel for many rows (paged_attn_tc.cu): rows per block, keys per tile.
constexpr int kTcRowsShift = 8;
constexpr int kTcRows = 1 << kTcRowsShift;
constexpr int kTcTileShift = 7;
constexpr int kTcTile = 1 << kTcTileShift;
int launch_tc(const Args& a, int64_t d, int ctas, cudaStream_t stream, const char* name);

// Tensor map of the pages as bf16 [pages * hkv * page_size, d], boxes of `box`
// rows x 64 columns with the 128-byte swizzle: 16-byte chunk c of a row r lands
// at chunk c ^ (r % 8) of its 128 bytes.
bool encode_pages(CUtensorMap* map, const void* pages, const Args& a, int d, int box);

// One box into shared memory, its bytes counted on `bar` (no multicast).
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(pipe::smem_u32(bar))
      : "memory");
}

// A worker's run of tiles.
struct Run {
  int64_t offset;  // into sequence s's tiles
  int64_t count;   // tiles; 0: nothing to do
  int64_t end;     // one past its last tile, counted over the whole batch
  int64_t share;   // tiles of every worker
  int s;
};

// Sums `v` over the CTA's threads below the caller (exclusive) and in all;
// `warps` holds one value per warp.  Whole CTA.
template <int THREADS>
__device__ __forceinline__ int64_t scan(int64_t v, int64_t* warps, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int64_t t = warps[w];
    if (w < warp) before += t;
    total += t;
  }
  __syncthreads();
  return before + x - v;
}

constexpr int kWarpSeqs = 128;  // sequences that a warp looks through by itself

// Tiles of sequence s, all its key heads.
__device__ __forceinline__ int64_t seq_work(const Args& a, int s) {
  return s < a.batch.s ? a.split.hkv * paged::head_work(a.split, paged::load_seq(a.batch, s)) : 0;
}

// The run of `worker`, for at most kWarpSeqs sequences, up to four a lane, whose
// tiles work_of(s) gives: no barrier between warps (whole warp).  Code that runs
// once is fetched cold, so it is kept short.
template <typename Work>
__device__ __forceinline__ Run warp_run(const Args& a, int worker, int workers,
                                        const Work& work_of) {
  const int lane = threadIdx.x & 31;
  const int per = (a.batch.s + 31) >> 5;
  const int first = lane * per;
  int64_t mine = 0;
#pragma unroll 1
  for (int i = 0; i < per; ++i) mine += work_of(first + i);
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
  Run run;
  run.share = paged::share_of(total, workers, a.least);
  const int64_t begin = run.share * worker;
  run.end = begin + run.share < total ? begin + run.share : total;
  run.count = run.end > begin ? run.end - begin : 0;
  run.offset = 0;
  run.s = 0;
  if (run.count == 0) return run;
  int64_t before = upto - mine;
  const int from = __ffs(__ballot_sync(0xffffffffu, before <= begin && begin < upto)) - 1;
  int s = first;
  if (lane == from) {
#pragma unroll 1
    for (; per > 1; ++s) {
      const int64_t next = before + work_of(s);
      if (begin < next) break;
      before = next;
    }
  }
  __syncwarp();
  run.s = __shfl_sync(0xffffffffu, s, from);
  run.offset = __shfl_sync(0xffffffffu, begin - before, from);
  return run;
}

// The runs of workers first .. first + N - 1, in runs[N] (shared memory), for
// any number of sequences.  Whole CTA of THREADS; up to THREADS sequences need
// one pass over the index arrays, longer batches two.
template <int THREADS, int N>
__device__ __forceinline__ void find_runs(const Args& a, int first, int workers, int64_t* warps,
                                          Run* runs) {
  const int tid = threadIdx.x;
  if (tid < N) runs[tid].count = 0;
  int64_t total = 0, mine = 0, before = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < a.batch.s; s0 += THREADS) {
    mine = seq_work(a, s0 + tid);
    int64_t sum;
    before = total + scan<THREADS>(mine, warps, sum);
    total += sum;
  }
  const int64_t share = paged::share_of(total, workers, a.least);
  if (share * first < total) {
    int64_t base = 0;
    for (int s0 = 0; s0 < a.batch.s; s0 += THREADS) {
      if (a.batch.s > THREADS) {
        mine = seq_work(a, s0 + tid);
        int64_t sum;
        before = base + scan<THREADS>(mine, warps, sum);
        base += sum;
      }
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
        const int64_t begin = share * (first + i);
        if (before <= begin && begin < before + mine) {
          const int64_t end = begin + share < total ? begin + share : total;
          runs[i] = Run{begin - before, end - begin, end, share, s0 + tid};
        }
      }
    }
  }
  __syncthreads();
}

// Reports a sequence with positions that the table has no room for (load_seq
// left them out).
__device__ __forceinline__ void check_length(const Args& a, int s, const paged::Seq& seq) {
  const int room = paged::capacity(a.batch);
  if (seq.len == room && a.batch.kv_len[s] > room) record_device_error(MOSS_ERR_VALUE);
}

// Slot of a cut piece.
__device__ __forceinline__ int slot_of(const paged::Piece& p, int worker) {
  return 2 * worker + (p.begins ? 1 : 0);
}
// Notes a cut piece that begins an item (others are found from it); it is the
// last of the worker's run.
__device__ __forceinline__ void note_piece(const Args& a, const paged::Piece& p,
                                           const paged::Range& r, const paged::Seq& seq,
                                           const Run& run, int worker) {
  if (!p.begins) return;
  Note n{};
  n.state = 1;
  n.last = static_cast<int>(
      paged::divide(run.end + (r.n - p.tile - p.n) - 1, run.share));
  n.h = p.h;
  n.row0 = seq.row0;
  n.block = p.block;
  const int rest = paged::rows_of(a.split, seq) - (p.block << a.split.rows_shift);
  n.rows = rest < (1 << a.split.rows_shift) ? rest : 1 << a.split.rows_shift;
  a.notes[worker] = n;
}
__device__ __forceinline__ void clear_note(const Args& a, int worker) {
  a.notes[worker].state = 0;
}

// Launched while the kernel before it may still run (each kernel waits for it
// before its first global access): the launch and the set-up cost nothing then.
template <typename... P, typename... V>
int launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                 const char* name, const V&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess)
    return fail(MOSS_ERR_CUDA, "%s: launch failed: %s", name, cudaGetErrorString(e));
  return launch_status(name);
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// A row's values are its sums times 1 / l; of a row that attends to nothing (l = 0)
// zeros, whatever the sums hold: a weight of zero times an infinity that other rows
// of the block attend to is NaN.
__device__ __forceinline__ float inverse_of(float l) {
  return l > 0.0f || l != l ? 1.0f / l : 0.0f;
}
__device__ __forceinline__ float normed(float sum, float inverse) {
  return inverse == 0.0f ? 0.0f : sum * inverse;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace pattn
}  // namespace moss
