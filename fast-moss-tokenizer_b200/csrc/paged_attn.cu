// Attention of a ragged batch of new tokens over a paged key/value history
// (sm_100a): the kernel for few query rows per key head, bound by the bytes
// of the keys and values, and the join of cut items.
//
//   out[t, h] = sum_p softmax_p(scale * q[t, h] . k[p]) v[p]
//   over the positions p of the token's sequence with p <= pos(t) and
//   p > pos(t) - context
//
// The query rows of one key head (tokens x query heads of the group) are
// packed into blocks of 8 or 16, the N of mma.sync.m16n8k16, with the keys of a
// 16-key step as its M: with so few rows the tensor cores' rate never matters
// (a step is 4 to 8 KB of HBM traffic and a few dozen small products), what
// matters is bytes in flight and how many steps are worked on at once.
//
// Every warp is a worker of its own: it takes an equal, contiguous run of
// 16-key groups (paged.cuh), crossing from item to item, and streams them
// through its own ring of shared-memory stages.  A group lies in one page
// (pages are multiples of 16 positions), so its keys and its values are one
// TMA box of 16 rows each (two for d = 128), requested by one lane.  The
// requests run ahead of the arithmetic by the whole ring, across items: the
// next item's page numbers are read while the current one streams.  No
// barrier between warps, no pipeline drain between items; ragged lengths,
// windows and one long history all keep every warp busy to the end.  Cut
// items are joined by a second small kernel, launched early (programmatic
// dependent launch).
//
// Measured: 61 single tokens over up to 8000 positions (32 heads over 8 of 128,
// 315 MB) 61 us, 5160 GB/s or 0.79 of a plain copy; one token over 131,000
// positions 94 us, 0.87; 64 streams of 4 tokens in a window of 250 (55 MB) 19 us,
// of which 6 until the first keys arrive and 9 steps of half a microsecond after
// them; one stream of 4 tokens over 2000 positions 13 us, the same latencies.
//
// The running maximum that the weights refer to moves only when a score
// exceeds it by more than 8 in base 2, so most steps need no exchange between
// the eight lanes of a row and no rescaling; the weights stay below 2^8.
//
// Rounding: scores, maxima, sums and outputs are float32.  The weights enter
// the second product as two bf16 terms, high + low (2^-16 relative): the
// tensor cores have time to spare here, and the result is then as close to
// the exact one as a float32 evaluation, up to the final rounding to bf16.
//
// Keys and values outside [lo, hi) of a block (past the history's end, or
// before every row's window) have no effect whatever those rows of a page
// hold: scores there are replaced, and rows of V overwritten with zeros in
// shared memory (a weight of zero does not silence an infinity).
#include <math_constants.h>

#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace moss {
namespace pattn {

constexpr int kGroupShift = 4;
constexpr int kGroup = 1 << kGroupShift;  // keys per step: the M of the MMAs
constexpr float kSlack = 8.0f;            // base-2 growth before a row is rescaled

// One stage: 16 keys, then 16 values, each as d / 64 boxes of 16 x 128 bytes.
constexpr uint32_t kBox = kGroup * 128;

// Warps of a CTA (one CTA per SM) and stages of a warp's ring: 192 KB in
// flight per SM, in as many warps as the registers allow (a step is a chain of
// dependent instructions, so warps in parallel are what hides it).
template <int D, int NT>
struct Shape {
  static constexpr int warps = D == 64 ? 16 : (NT == 1 ? 12 : 8);
  static constexpr int stages = D == 64 ? 3 : (NT == 1 ? 2 : 3);
  static constexpr uint32_t half = kBox * (D / 64);
  static constexpr uint32_t ring = stages * 2 * half;
  static constexpr size_t smem = 1024 + static_cast<size_t>(warps) * ring;
};

struct RowsArgs {
  CUtensorMap k_map;  // box {64, 16}
  CUtensorMap v_map;
  Args a;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The transpose of an 8 x 8 matrix of 16-bit values held by the warp (row
// lane / 4, columns 2 (lane % 4) and + 1).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte chunk c of row r of a stage's keys or values, as the TMA leaves it.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return static_cast<uint32_t>((c >> 3) * kBox + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// What a warp's requests leave for its arithmetic about a piece.
struct Job {
  paged::Seq seq;
  paged::Piece p;
  paged::Range r;
  int g, steps;  // first group and groups (an empty piece: one step without data)
};
constexpr int kJobs = 8;  // more than the stages of a ring and the piece ahead

template <int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::warps * 32, 1)
    rows_kernel(const __grid_constant__ RowsArgs args) {
  using S = Shape<D, NT>;
  constexpr int kWarps = S::warps, kStages = S::stages;
  constexpr uint32_t kHalf = S::half;
  constexpr int kRows = 8 * NT;
  constexpr int kKs = D / 16;  // k-steps of k.q, 16-row tiles of the output's transpose
  static_assert(kStages + 3 <= kJobs, "a job outlives the steps requested for it");
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long bars[kWarps][kStages];
  __shared__ int64_t scan_smem[kWarps], works[kWarpSeqs];
  __shared__ Run runs[kWarps];
  __shared__ paged::Walker walkers[kWarps];
  __shared__ Job jobs_smem[kWarps][kJobs];
  const Args& a = args.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int workers = gridDim.x * kWarps, worker = blockIdx.x * kWarps + warp;
  unsigned long long* full = bars[warp];
  Job* jobs = jobs_smem[warp];
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) pipe::mbar_init(&full[i], 1);
    pipe::fence_mbar_init();
    prefetch_map(&args.k_map);
    prefetch_map(&args.v_map);
  }
  __syncwarp();
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  if (lane == 0) clear_note(a, worker);
  Run run;
  // One sequence a lane needs no word between warps; of more, a thread looks at
  // one for the whole CTA (64 streams in a window of 250 19.8 us, 20.4 where
  // every lane looks at two; one stream 12.8, 13.1 with the barrier).
  if (a.batch.s <= 32) {
    run = warp_run(a, worker, workers, [&](int s) { return seq_work(a, s); });
  } else if (a.batch.s <= kWarpSeqs) {
    if (static_cast<int>(threadIdx.x) < kWarpSeqs) works[threadIdx.x] = seq_work(a, threadIdx.x);
    __syncthreads();
    run = warp_run(a, worker, workers, [&](int s) { return works[s]; });
  } else {
    find_runs<kWarps * 32, kWarps>(a, blockIdx.x * kWarps, workers, scan_smem, runs);
    run = runs[warp];
  }
  if (run.count == 0) return;
  unsigned char* ring =
      smem_raw + ((1024u - (pipe::smem_u32(smem_raw) & 1023u)) & 1023u) + warp * S::ring;
  const uint32_t ring_u = pipe::smem_u32(ring);
  const int shift = a.batch.page_shift, page_mask = (1 << shift) - 1;
  const int group = static_cast<int>(a.split.group.d);

  // ---- requests.  The walker lives in shared memory between pieces; the
  // page numbers of the piece ahead are loaded while the current one streams.
  {
    paged::Walker w;
    w.start(a.batch, a.split, run.s, run.offset, run.count);
    if (lane == 0) walkers[warp] = w;
    __syncwarp();
  }
  int made = 0;      // jobs written
  bool more_jobs = true;
  int ahead_ids = 0, ahead_more = 0;  // of the newest job
  auto ids_at = [&](const int32_t* table, int g, int end) {
    return g + lane < end ? table[((g + lane) << kGroupShift) >> shift] : 0;
  };
  auto make_job = [&] {
    paged::Walker w = walkers[warp];
    __syncwarp();
    Job job;
    more_jobs = w.next(a.batch, a.split, job.p, job.r);
    if (!more_jobs) return;
    job.seq = w.seq;
    job.g = job.r.tile0 + job.p.tile;
    job.steps = job.p.n;
    if (lane == 0) {
      check_length(a, job.p.s, job.seq);
      walkers[warp] = w;
      jobs[made % kJobs] = job;
    }
    ++made;
    __syncwarp();
    const int32_t* table = a.batch.table + static_cast<int64_t>(job.p.s) * a.batch.max_pages;
    const int end = job.r.hi > job.r.lo ? job.g + job.steps : job.g;
    ahead_ids = ids_at(table, job.g, end);
    ahead_more = ids_at(table, job.g + 32, end);
  };
  // the job being requested
  const int32_t* table = nullptr;
  int job_in = -1, g = 0, g_end = 0, g_first = 0, head = 0, ids = 0, ids_more = 0;
  bool empty_job = false;
  int issued = 0, stage_in = 0;
  make_job();
  auto request = [&] {
    if (g == g_end) {
      if (job_in + 1 == made) return;
      ++job_in;
      const Job& job = jobs[job_in % kJobs];
      table = a.batch.table + static_cast<int64_t>(job.p.s) * a.batch.max_pages;
      g = g_first = job.g;
      g_end = g + job.steps;
      head = job.p.h;
      empty_job = job.r.hi <= job.r.lo;
      ids = ahead_ids;
      ids_more = ahead_more;
      if (more_jobs) make_job();
    }
    const int i = g - g_first;
    if (i > 0 && (i & 31) == 0) {
      ids = ids_more;
      ids_more = ids_at(table, g + 32, g_end);
    }
    const int page = __shfl_sync(0xffffffffu, ids, i & 31);
    if (lane == 0) {
      unsigned long long* bar = &full[stage_in];
      if (!empty_job && page >= 0 && page < a.batch.pages) {
        const int y = ((page * a.split.hkv + head) << shift) + ((g << kGroupShift) & page_mask);
        const uint32_t dst = ring_u + stage_in * 2 * kHalf;
        pipe::mbar_arrive_expect_tx(bar, 2 * kHalf);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_load(dst + c * kBox, &args.k_map, c * 64, y, bar);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load(dst + kHalf + c * kBox, &args.v_map, c * 64, y, bar);
      } else {
        if (!empty_job) record_device_error(MOSS_ERR_VALUE);
        pipe::mbar_arrive(bar);
      }
    }
    ++g;
    ++issued;
    if (++stage_in == kStages) stage_in = 0;
  };
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) request();

  // ---- arithmetic.  Scores and output are held transposed (keys x queries,
  // d x queries): the 8 (or 16) query rows are the MMAs' N.
  const int row = lane >> 2, pair = (lane & 3) * 2;
  int done = 0, stage = 0, phase = 0;
  bool ok = true;
#pragma unroll 1
  for (int at_job = 0; ok && at_job < made; ++at_job) {
    const Job& job = jobs[at_job % kJobs];
    const paged::Seq seq = job.seq;
    const int h = job.p.h;
    const int r0 = job.p.block * kRows;
    const int rest = paged::rows_of(a.split, seq) - r0;
    const int rows = rest < kRows ? rest : kRows;
    const int lo = job.r.lo, hi = job.r.hi;
    const int steps = job.steps, g0 = job.g;
    // query fragments: row lane / 4 of each tile of 8
    uint32_t qf[NT][kKs][2];
    int64_t row_at[NT];          // the row's place in q and out
    int low[NT][2], pos[NT][2];  // keys [low, pos] are query pair + e's
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + 8 * nt + row;
      const int t = paged::quotient(r, a.split.group);
      row_at[nt] = ((static_cast<int64_t>(seq.row0) + t) * a.hq + h * group + (r - t * group)) * D;
      const bool on = 8 * nt + row < rows;
      const uint16_t* src = a.q + row_at[nt] + pair;
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) {
        qf[nt][ks][0] = on ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
        qf[nt][ks][1] = on ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pos[nt][e] =
            seq.len - seq.t + paged::quotient(r0 + 8 * nt + pair + e, a.split.group);
        low[nt][e] = paged::window_start(pos[nt][e], a.split.context);
      }
    }
    // groups inside [the last row's window start, the first row's position]
    // need no mask
    const int free_from = paged::window_start(
        seq.len - seq.t + paged::quotient(r0 + rows - 1, a.split.group), a.split.context);
    const int free_to = seq.len - seq.t + paged::quotient(r0, a.split.group);

    float o[kKs][NT][4];
#pragma unroll
    for (int i = 0; i < kKs; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
    float m[NT][2], l[NT][2];  // base 2, scaled; this lane's part of the sum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -CUDART_INF_F;
      l[nt][0] = l[nt][1] = 0.0f;
    }

#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      // one lane asks: the barrier serves its callers one by one
      if (lane == 0) ok = pipe::mbar_wait(&full[stage], phase);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      if (hi > lo) {
        const uint32_t kst = ring_u + stage * 2 * kHalf;
        const uint32_t vst = kst + kHalf;
        const int at = (g0 + step) << kGroupShift;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
          uint32_t k[4];
          // matrices: keys 0-7, 8-15 ((lane >> 3) & 1), dims 16 ks + 8 (lane >> 4)
          ldmatrix4(k, kst + chunk_at((lane & 7) + (((lane >> 3) & 1) << 3),
                                      ks * 2 + (lane >> 4)));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(s[nt], k, qf[nt][ks][0], qf[nt][ks][1]);
        }
        if (at < free_from || at + kGroup - 1 > free_to) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = at + row + (e >> 1) * 8;
              if (key < low[nt][e & 1] || key > pos[nt][e & 1]) s[nt][e] = -CUDART_INF_F;
            }
          // rows of V that no row of the block attends to
          if (at < lo || at + kGroup > hi) {
            for (int i = lane; i < kGroup * (D / 8); i += 32) {
              const int r = i & (kGroup - 1), c = i >> kGroupShift;
              if (at + r < lo || at + r >= hi)
                *reinterpret_cast<uint4*>(ring + stage * 2 * kHalf + kHalf + chunk_at(r, c)) =
                    make_uint4(0, 0, 0, 0);
            }
            // before the stage's next copy, and the reads below
            tc::fence_async_shared();
            __syncwarp();
          }
        }
        float top[NT][2];
        bool move = false;  // -inf against -inf is no move
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[nt][e] = fmaxf(s[nt][e], s[nt][e + 2]) * a.scale2;
            move |= top[nt][e] - m[nt][e] > kSlack;
          }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = top[nt][e];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
              const float now = fmaxf(m[nt][e], x);
              const float keep = now == -CUDART_INF_F ? 1.0f : exp2_fast(m[nt][e] - now);
              m[nt][e] = now;
              l[nt][e] *= keep;
#pragma unroll
              for (int i = 0; i < kKs; ++i) {
                o[i][nt][e] *= keep;
                o[i][nt][e + 2] *= keep;
              }
            }
        }
        uint32_t hi_p[NT][2], lo_p[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // a row with no key yet keeps weight 0 throughout
          const float base0 = m[nt][0] == -CUDART_INF_F ? 0.0f : m[nt][0];
          const float base1 = m[nt][1] == -CUDART_INF_F ? 0.0f : m[nt][1];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float e0 = exp2_fast(fmaf(s[nt][2 * j], a.scale2, -base0));
            const float e1 = exp2_fast(fmaf(s[nt][2 * j + 1], a.scale2, -base1));
            l[nt][0] += e0;
            l[nt][1] += e1;
            const uint32_t x = pack_bf16x2(e0, e1);
            hi_p[nt][j] = transpose8(x);
            lo_p[nt][j] = transpose8(pack_bf16x2(e0 - __uint_as_float(x << 16),
                                                 e1 - __uint_as_float(x & 0xffff0000u)));
          }
        }
#pragma unroll
        for (int i = 0; i < kKs; ++i) {
          uint32_t v[4];
          // matrices: keys 0-7, 8-15 (lane >> 4), dims 16 i + 8 ((lane >> 3) & 1)
          ldmatrix4_trans(v, vst + chunk_at((lane & 7) + ((lane >> 4) << 3),
                                            i * 2 + ((lane >> 3) & 1)));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(o[i][nt], v, hi_p[nt][0], hi_p[nt][1]);
            mma16816(o[i][nt], v, lo_p[nt][0], lo_p[nt][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      request();
      ++done;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok) break;

    // ---- the piece's rows
    const bool whole = job.p.whole;
    const int64_t slot_row = static_cast<int64_t>(whole ? 0 : slot_of(job.p, worker)) * kRows;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
      if (whole) {
        const float inv[2] = {inverse_of(l[nt][0]), inverse_of(l[nt][1])};
#pragma unroll
        for (int i = 0; i < kKs; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = transpose8(
                pack_bf16x2(normed(o[i][nt][2 * j], inv[0]), normed(o[i][nt][2 * j + 1], inv[1])));
            if (8 * nt + row < rows)
              *reinterpret_cast<uint32_t*>(a.out + row_at[nt] + i * 16 + j * 8 + pair) = x;
          }
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * nt + pair + e;
          if (r < rows) {
            float* dst = a.partial + (slot_row + r) * D + row;
#pragma unroll
            for (int i = 0; i < kKs; ++i) {
              dst[i * 16] = o[i][nt][e];
              dst[i * 16 + 8] = o[i][nt][e + 2];
            }
            if (row == 0) a.stats[slot_row + r] = make_float2(m[nt][e], l[nt][e]);
          }
        }
      }
    }
    if (!whole && lane == 0) note_piece(a, job.p, job.r, seq, run, worker);
    __syncwarp();  // the job's slot may be written again
  }
  // after a wait that gave up: copies still in flight land before the CTA retires
  for (; !ok && done < issued; ++done) {
    pipe::mbar_wait(&full[stage], phase);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
}

// Joins the pieces of every cut item, in a fixed order (results do not vary).
// A warp looks at one worker's note and joins what that worker began; an item
// of many pieces (a long history spread over the device) is left to the whole
// block, whose warps take every eighth piece each and add up in shared memory.
// blockIdx.y takes join_rows of an item's rows.
//
// What costs here is latency, not bytes: a batch of pieces is loaded at once,
// statistics and values together, before any of it is used.
constexpr int kJoinWarps = 8;
constexpr int kJoinThreads = kJoinWarps * 32;
constexpr int kManyPieces = 9;
constexpr int kBatch = 4;

struct Sum {
  float4 v;
  float top, l;
};

template <int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Args a,
                                                            int workers, int join_rows) {
  constexpr int kCols = D / 4;         // float4 of a row
  constexpr int kPer = 32 / kCols;     // rows a warp takes at a time
  __shared__ Sum sums[kJoinWarps][32];
  __shared__ Note notes[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = lane % kCols, sub = lane / kCols;
  const int group = static_cast<int>(a.split.group.d);
  const int from = blockIdx.y * join_rows;
  cudaGridDependencySynchronize();
  // Pieces k0, k0 + step, ... below `count` of row r, column col.
  auto collect = [&](int first, int count, int k0, int step, int r) {
    Sum sum;
    sum.v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    sum.top = -CUDART_INF_F;
    sum.l = 0.0f;
    for (int base = k0; base < count; base += kBatch * step) {
      float2 st[kBatch];
      float4 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int k = base + i * step;
        st[i] = make_float2(-CUDART_INF_F, 0.0f);
        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < count) {
          const int64_t at =
              (static_cast<int64_t>(2 * (first + k) + (k == 0 ? 1 : 0)) << a.split.rows_shift) + r;
          st[i] = a.stats[at];
          v[i] = *reinterpret_cast<const float4*>(a.partial + at * D + col * 4);
        }
      }
      float now = sum.top;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) now = fmaxf(now, st[i].x);
      const float shift = now == -CUDART_INF_F ? 0.0f : now;
      const float keep = exp2_fast(sum.top - shift);
      sum.top = now;
      sum.l *= keep;
      sum.v.x *= keep;
      sum.v.y *= keep;
      sum.v.z *= keep;
      sum.v.w *= keep;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float g = exp2_fast(st[i].x - shift);
        sum.l = fmaf(st[i].y, g, sum.l);
        sum.v.x = fmaf(v[i].x, g, sum.v.x);
        sum.v.y = fmaf(v[i].y, g, sum.v.y);
        sum.v.z = fmaf(v[i].z, g, sum.v.z);
        sum.v.w = fmaf(v[i].w, g, sum.v.w);
      }
    }
    return sum;
  };
  auto put = [&](const Note& n, const Sum& sum, int r) {
    const float inv = inverse_of(sum.l);
    const int rr = (n.block << a.split.rows_shift) + r;
    const int t = paged::quotient(rr, a.split.group);
    uint16_t* dst = a.out + ((static_cast<int64_t>(n.row0) + t) * a.hq + n.h * group +
                             (rr - t * group)) * D + col * 4;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_bf16x2(normed(sum.v.x, inv), normed(sum.v.y, inv)),
                   pack_bf16x2(normed(sum.v.z, inv), normed(sum.v.w, inv)));
  };
  auto pieces_of = [&](const Note& n, int first) {
    return n.state == 0 || n.last < first || n.last >= workers ? 0 : n.last - first + 1;
  };
  const int mine = blockIdx.x * kJoinWarps + warp;
  Note n{};
  if (mine < workers) n = a.notes[mine];
  const int pieces = pieces_of(n, mine);
  const int to = from + join_rows < n.rows ? from + join_rows : n.rows;
  if (pieces > 0 && pieces < kManyPieces) {
    for (int r = from + sub; r < to; r += kPer) put(n, collect(mine, pieces, 0, 1, r), r);
  }
  if (!__syncthreads_or(pieces >= kManyPieces)) return;
  if (lane == 0) notes[warp] = n;
  __syncthreads();
  for (int w = 0; w < kJoinWarps; ++w) {
    const Note big = notes[w];
    const int first = blockIdx.x * kJoinWarps + w;
    const int count = pieces_of(big, first);
    if (count < kManyPieces) continue;
    const int end = from + join_rows < big.rows ? from + join_rows : big.rows;
    for (int r = from; r < end; r += kPer) {
      const Sum sum = collect(first, count, warp, kJoinWarps, r + sub < end ? r + sub : r);
      sums[warp][lane] = sum;
      __syncthreads();
      if (warp == 0 && r + sub < end) {
        float top = sum.top;
#pragma unroll
        for (int k = 1; k < kJoinWarps; ++k) top = fmaxf(top, sums[k][lane].top);
        const float shift = top == -CUDART_INF_F ? 0.0f : top;
        Sum all;
        all.v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        all.top = top;
        all.l = 0.0f;
#pragma unroll
        for (int k = 0; k < kJoinWarps; ++k) {
          const Sum part = sums[k][lane];
          const float g = exp2_fast(part.top - shift);
          all.l = fmaf(part.l, g, all.l);
          all.v.x = fmaf(part.v.x, g, all.v.x);
          all.v.y = fmaf(part.v.y, g, all.v.y);
          all.v.z = fmaf(part.v.z, g, all.v.z);
          all.v.w = fmaf(part.v.w, g, all.v.w);
        }
        put(big, all, r + sub);
      }
      __syncthreads();
    }
  }
}

// Workspace: a note a worker, stats and partial rows of two slots a worker.
struct Space {
  int64_t notes, stats, partial, total;  // byte offsets
};
Space space(int64_t workers, int64_t rows, int64_t d) {
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  Space s;
  s.notes = 0;
  s.stats = up(workers * static_cast<int64_t>(sizeof(Note)));
  s.partial = s.stats + up(2 * workers * rows * static_cast<int64_t>(sizeof(float2)));
  s.total = s.partial + 2 * workers * rows * d * static_cast<int64_t>(sizeof(float));
  return s;
}
void place(Args& a, void* workspace, const Space& s) {
  unsigned char* w = static_cast<unsigned char*>(workspace);
  a.notes = reinterpret_cast<Note*>(w + s.notes);
  a.stats = reinterpret_cast<float2*>(w + s.stats);
  a.partial = reinterpret_cast<float*>(w + s.partial);
}

// Query rows per key head above which a sequence goes to the tensor-memory
// kernel, whose blocks of 256 rows cost the same however few are used: 64
// streams of 24 rows in a window of 250 37 us here, 77 there, of 64 rows 62 and
// 87; 16 streams of 32 rows over 2000 keys 69 and 68, of 64 rows 106 and 73.  The
// border is also where the weights go from two bf16 terms to one, so it looks at
// the sequence's own rows, not at its neighbours: a sequence by itself is in part
// faster there from 16 rows on (32 rows over 2000 keys 17 us here, 15 there, over
// 30,000 56 and 53; 16 rows 17 and 15, 42 and 53).  Rows are only half of what
// parts the kernels in time, keys a block the other: in a short window 64 rows are
// still faster here, over long histories 32 already there.
constexpr int kFewRows = 32;
// Rows for which the narrow form of the kernel (8 rows a block, more warps) is
// taken: 4 rows in a window of 250 20 us, 24 in the wide form.
constexpr int kNarrowRows = 8;
// Groups that a warp takes at least.  A group more is half a microsecond, a
// piece more in the join less: one stream of 4 tokens over 2000 keys 12.8, 13.2,
// 13.9, 15.4 us for 2, 3, 4, 6.
constexpr int kLeastGroups = 2;
// What an item costs before its keys (paged::Split::setup), in groups, and a
// block of many rows in tiles.  Measured without, with these, and with three
// times as much: 64 streams in a window of 250 26.0, 20.3, 20.6 us; prompts
// beside single tokens 107, 79, 90 us (later 78, 74, 76 for 2, 3, 4 tiles).
constexpr int kSetupGroups = 2;
constexpr int kTcSetup = 3;

template <int D>
int launch_join(const Args& a, int workers, cudaStream_t stream, const char* name) {
  // rows side by side in blocks of their own: one row's latency, not the sum
  const int rows = 1 << a.split.rows_shift;
  const int join_rows = 128 / D;
  const dim3 grid(static_cast<unsigned>((workers + kJoinWarps - 1) / kJoinWarps),
                  static_cast<unsigned>(rows / join_rows), 1);
  return launch_early(join_kernel<D>, grid, kJoinThreads, 0, stream, name, a, workers, join_rows);
}

template <int D, int NT>
int launch_rows(Args& a, void* workspace, cudaStream_t stream, const char* name) {
  using S = Shape<D, NT>;
  const int ctas = sm_count();
  const int workers = ctas * S::warps;
  a.split.rows_shift = NT == 1 ? 3 : 4;
  a.split.tile_shift = kGroupShift;
  a.split.setup = kSetupGroups;
  a.least = kLeastGroups + kSetupGroups;
  place(a, workspace, space(workers, 8 * NT, D));
  RowsArgs args{};
  args.a = a;
  if (!encode_pages(&args.k_map, a.k_pages, a, D, kGroup) ||
      !encode_pages(&args.v_map, a.v_pages, a, D, kGroup))
    return fail(MOSS_ERR_CUDA, "%s: tensor map encoding failed", name);
  static bool configured[kMaxDevices] = {};
  allow_dynamic_smem(rows_kernel<D, NT>, S::smem, configured);
  const int status = launch_early(rows_kernel<D, NT>, dim3(static_cast<unsigned>(ctas), 1, 1),
                                  S::warps * 32, S::smem, stream, name, args);
  return status != MOSS_OK ? status : launch_join<D>(a, workers, stream, name);
}

// most: bound of the rows per key head of any sequence.  Sequences of few rows
// and longer ones each have their kernel; where the bound allows both, both run
// and each takes its own.  A single sequence has one kind only, the bound's.
template <int D>
int run(Args& a, int64_t most, void* workspace, cudaStream_t stream,
        const char* name) {
  const bool many = most > kFewRows;
  const bool few = !many || a.batch.s > 1;
  int status = MOSS_OK;
  if (few) {
    a.split.min_q = 1;
    a.split.max_q = many ? kFewRows : 0x7fffffff;
    status = most <= kNarrowRows ? launch_rows<D, 1>(a, workspace, stream, name)
                       : launch_rows<D, 2>(a, workspace, stream, name);
  }
  if (many && status == MOSS_OK) {
    const int ctas = sm_count();
    a.split.rows_shift = kTcRowsShift;
    a.split.tile_shift = kTcTileShift;
    a.split.min_q = few ? kFewRows + 1 : 1;
    a.split.max_q = 0x7fffffff;
    a.split.setup = kTcSetup;
    a.least = 1 + kTcSetup;  // a tile at least
    place(a, workspace, space(ctas, kTcRows, D));
    status = launch_tc(a, D, ctas, stream, name);
  }
  return status;
}

template <int D>
int64_t workspace_bytes(bool many) {
  const int64_t one = space(sm_count() * Shape<D, 1>::warps, 8, D).total;
  const int64_t two = space(sm_count() * Shape<D, 2>::warps, 16, D).total;
  const int64_t tc = many ? space(sm_count(), kTcRows, D).total : 0;
  const int64_t few = one > two ? one : two;
  return few > tc ? few : tc;
}

}  // namespace pattn
}  // namespace moss

using namespace moss;

extern "C" int64_t moss_paged_attention_workspace(int64_t d, int64_t rows) {
  if (d != 64 && d != 128) return 0;
  const bool many = rows > pattn::kFewRows;
  return d == 64 ? pattn::workspace_bytes<64>(many) : pattn::workspace_bytes<128>(many);
}

extern "C" int moss_paged_attention(const void* q, const void* k_pages, const void* v_pages,
                                    const int64_t* q_start, const int64_t* kv_len,
                                    const int32_t* page_table, int64_t n, int64_t s, int64_t hq,
                                    int64_t hkv, int64_t d, int64_t pages, int64_t page_size,
                                    int64_t max_pages, int64_t max_tokens, int64_t context,
                                    float scale, void* workspace, int64_t workspace_bytes,
                                    void* out, void* stream) {
  const char* name = "moss_paged_attention";
  if (n < 0 || s < 0 || hq < 1 || hkv < 1 || hq % hkv || d < 1 || pages < 0 || max_pages < 0 ||
      max_tokens < 0 || context < 0)
    return fail(MOSS_ERR_VALUE, "%s: bad shape", name);
  if (!(scale > 0.0f) || !isfinite(scale))
    return fail(MOSS_ERR_VALUE, "%s: scale must be positive and finite", name);
  if (d != 64 && d != 128) return fail(MOSS_ERR_UNSUPPORTED, "%s: heads of 64 or 128", name);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return fail(MOSS_ERR_UNSUPPORTED, "%s: pages of 16, 32, 64, 128 or 256 positions", name);
  if (n == 0 || s == 0) return MOSS_OK;
  if (!q || !k_pages || !v_pages || !q_start || !kv_len || !page_table || !out || !workspace)
    return fail(MOSS_ERR_VALUE, "%s: null pointer", name);
  if (n > 0x3fffffff / (hq / hkv) || s > 0x3fffffff || hq > (1 << 20) || pages > 0x7fffffff ||
      max_pages > 0x7ffffeff / page_size || pages > 0x7fffffff / (hkv * page_size))
    return fail(MOSS_ERR_UNSUPPORTED, "%s: too large", name);
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      !aligned16(workspace))
    return fail(MOSS_ERR_VALUE, "%s: buffers must be 16-byte aligned", name);
  const int64_t group = hq / hkv;
  const int64_t most = (max_tokens > 0 && max_tokens < n ? max_tokens : n) * group;
  if (workspace_bytes < moss_paged_attention_workspace(d, most))
    return fail(MOSS_ERR_VALUE, "%s: the workspace is too small", name);
  pattn::Args a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k_pages = static_cast<const uint16_t*>(k_pages);
  a.v_pages = static_cast<const uint16_t*>(v_pages);
  a.out = static_cast<uint16_t*>(out);
  a.batch.q_start = q_start;
  a.batch.kv_len = kv_len;
  a.batch.table = page_table;
  a.batch.n = static_cast<int>(n);
  a.batch.s = static_cast<int>(s);
  a.batch.max_pages = static_cast<int>(max_pages);
  a.batch.pages = static_cast<int>(pages);
  while ((1 << a.batch.page_shift) < page_size) ++a.batch.page_shift;
  a.split.group = make_fastdiv(static_cast<uint32_t>(hq / hkv));
  a.split.hkv = static_cast<int>(hkv);
  a.split.context = context == 0 || context > 0x7fffffff ? 0x7fffffff
                                                         : static_cast<int>(context);
  a.split.min_q = 1;
  a.split.max_q = 0x7fffffff;
  a.hq = static_cast<int>(hq);
  a.scale2 = scale * 1.4426950408889634f;
  return d == 64 ? pattn::run<64>(a, most, workspace, as_stream(stream), name)
                 : pattn::run<128>(a, most, workspace, as_stream(stream), name);
}

extern "C" int64_t moss_paged_attention_plan(const int64_t* q_start, const int64_t* kv_len,
                                             int64_t n, int64_t s, int64_t group, int64_t hkv,
                                             int64_t page_size, int64_t max_pages, int64_t context,
                                             int64_t rows, int64_t tile, int64_t setup,
                                             int64_t ctas, int64_t* pieces, int64_t max_pieces) {
  if (!q_start || !kv_len || !pieces || n < 0 || s < 0 || group < 1 || hkv < 1 || rows < 1 ||
      tile < 1 || setup < 0 || (rows & (rows - 1)) || (tile & (tile - 1)) || ctas < 1 ||
      page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return -1;
  // as moss_paged_attention, whose index arithmetic this is
  if (group > (1 << 20) || hkv > (1 << 20) / group || n > 0x3fffffff / group || s > 0x3fffffff ||
      max_pages < 0 || max_pages > 0x7ffffeff / page_size || context < 0 || rows > (1 << 20) ||
      tile > (1 << 20) || setup > (1 << 20) || ctas > (1 << 24))
    return -1;
  paged::Batch b{};
  b.q_start = q_start;
  b.kv_len = kv_len;
  b.n = static_cast<int>(n);
  b.s = static_cast<int>(s);
  b.max_pages = static_cast<int>(max_pages);
  while ((1 << b.page_shift) < page_size) ++b.page_shift;
  paged::Split w{};
  while ((1 << w.rows_shift) < rows) ++w.rows_shift;
  while ((1 << w.tile_shift) < tile) ++w.tile_shift;
  w.group = make_fastdiv(static_cast<uint32_t>(group));
  w.hkv = static_cast<int>(hkv);
  w.context = context == 0 || context > 0x7fffffff ? 0x7fffffff : static_cast<int>(context);
  w.min_q = 1;
  w.max_q = 0x7fffffff;
  w.setup = static_cast<int>(setup);
  int64_t total = 0;
  for (int i = 0; i < b.s; ++i) total += hkv * paged::head_work(w, paged::load_seq(b, i));
  const int least = (tile == pattn::kGroup ? pattn::kLeastGroups : 1) + w.setup;
  const int64_t share = paged::share_of(total, static_cast<int>(ctas), least);
  int64_t count = 0;
  for (int64_t c = 0; c < ctas; ++c) {
    const int64_t begin = share * c;
    const int64_t end = begin + share < total ? begin + share : total;
    if (begin >= end) break;
    int64_t before = 0;
    int i = 0;
    for (;; ++i) {
      const int64_t mine = hkv * paged::head_work(w, paged::load_seq(b, i));
      if (begin < before + mine) break;
      before += mine;
    }
    paged::Walker walk;
    walk.start(b, w, i, begin - before, end - begin);
    paged::Piece p;
    paged::Range r;
    while (walk.next(b, w, p, r)) {
      if (count < max_pieces) {
        int64_t* o = pieces + count * 9;
        o[0] = c;
        o[1] = p.s;
        o[2] = p.h;
        o[3] = p.block;
        o[4] = p.tile;
        o[5] = p.n;
        o[6] = r.lo;
        o[7] = r.hi;
        o[8] = (p.begins ? 1 : 0) + (p.ends ? 2 : 0);
      }
      ++count;
    }
  }
  return count;
}
