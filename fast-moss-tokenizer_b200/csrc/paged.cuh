// Geometry of the paged key/value history shared by its kernels: where a
// position lives, which keys a block of query rows reads, and how the work
// of a ragged batch is split over a persistent grid.
//
// Positions of sequence s live in pages of a pool [pages, kv_heads,
// page_size, d]: position p in page table[s, p / page_size], row p %
// page_size.  The new tokens of all sequences are packed row after row;
// sequence s owns rows q_start[s] .. q_start[s + 1] - 1, and they are its
// last positions: kv_len[s] - T .. kv_len[s] - 1.
//
// Everything here is host and device code, so that the bounds and the split
// can be checked on the CPU (moss_paged_attention_plan).
#pragma once

#include "common.cuh"

namespace moss {
namespace paged {

struct Batch {
  const int64_t* q_start;  // [s + 1]
  const int64_t* kv_len;   // [s]
  const int32_t* table;    // [s, max_pages]
  int n;                   // packed rows
  int s;                   // sequences
  int max_pages;           // columns of the table
  int pages;               // pages of the pool
  int page_shift;          // log2(page_size)
};

// Positions one sequence can hold (below 2^31: checked on the host).
__host__ __device__ inline int capacity(const Batch& b) { return b.max_pages << b.page_shift; }

struct Seq {
  int row0;  // first packed row
  int t;     // new tokens
  int len;   // positions, the new tokens included
};

// The sequence's rows and length, clamped so that nothing later leaves the
// buffers whatever the device arrays hold.  Of rows that pass the packed ones
// those that are there keep their positions.
__host__ __device__ inline Seq load_seq(const Batch& b, int s) {
  int64_t r0 = b.q_start[s], r1 = b.q_start[s + 1], len = b.kv_len[s];
  len = (len < 0 ? 0 : len) - (r1 > b.n ? r1 - b.n : 0);
  r0 = r0 < 0 ? 0 : (r0 > b.n ? b.n : r0);
  r1 = r1 < r0 ? r0 : (r1 > b.n ? b.n : r1);
  const int64_t cap = capacity(b);
  len = len < 0 ? 0 : (len > cap ? cap : len);
  return Seq{static_cast<int>(r0), static_cast<int>(r1 - r0), static_cast<int>(len)};
}

// Quotient of x >= 0 by a run-time constant.
__host__ __device__ inline int quotient(int x, const FastDiv& f) {
#ifdef __CUDA_ARCH__
  return static_cast<int>(fast_div(static_cast<uint32_t>(x), f));
#else
  return static_cast<int>(static_cast<uint32_t>(x) / f.d);
#endif
}

// Work split of the attention.  Query rows of one key head are packed token
// by token (row = token * group + query head of the group) and cut into
// blocks of 2^rows_shift; an item is (sequence, key head, block) and its work
// the number of 2^tile_shift-key tiles it reads.
struct Split {
  int rows_shift;     // query rows per block
  int tile_shift;     // keys per tile
  int hkv;            // key heads
  int context;        // window in positions (INT32_MAX: none)
  int min_q, max_q;   // only sequences with min_q <= t * group <= max_q
  int setup;          // what starting an item costs, in tiles (see Walker)
  FastDiv group;      // query heads per key head
};

struct Range {
  int lo, hi;      // keys read by the block: [lo, hi), empty when hi <= lo
  int tile0, n;    // first tile and number of tiles (at least one)
};

// First position that the row at position `pos` attends to (if any).
__host__ __device__ inline int window_start(int pos, int context) {
  return pos >= context ? pos - context + 1 : 0;
}

// Rows of a key head; t * group < 2^30 (checked on the host).
__host__ __device__ inline int rows_of(const Split& w, const Seq& q) {
  return q.t * static_cast<int>(w.group.d);
}

__host__ __device__ inline int row_blocks(const Split& w, const Seq& q) {
  const int rows = rows_of(w, q);
  if (rows < w.min_q || rows > w.max_q) return 0;
  return (rows + (1 << w.rows_shift) - 1) >> w.rows_shift;
}

__host__ __device__ inline Range block_range(const Split& w, const Seq& q, int block) {
  const int all = rows_of(w, q);
  const int r0 = block << w.rows_shift;
  const int r1 = all - r0 < (1 << w.rows_shift) ? all : r0 + (1 << w.rows_shift);
  const int first = q.len - q.t + quotient(r0, w.group);       // position of the first row
  const int last = q.len - q.t + quotient(r1 - 1, w.group);    // and of the last
  Range r;
  r.lo = window_start(first, w.context);
  r.hi = last + 1;
  if (r.hi <= r.lo) {  // no key at all: one empty tile still writes the rows
    r.lo = r.hi = 0;
    r.tile0 = 0;
    r.n = 1;
    return r;
  }
  r.tile0 = r.lo >> w.tile_shift;
  r.n = ((r.hi - 1) >> w.tile_shift) + 1 - r.tile0;
  return r;
}

// Tiles of one key head of a sequence.
__host__ __device__ inline int64_t head_work(const Split& w, const Seq& q) {
  const int blocks = row_blocks(w, q);
  int64_t sum = 0;
#ifdef __CUDA_ARCH__
#pragma unroll 1
#endif
  for (int b = 0; b < blocks; ++b) sum += block_range(w, q, b).n + w.setup;
  return sum;
}

// a / b for a >= 0, b > 0: a 64-bit division costs hundreds of instructions on
// the device and is hardly ever needed.
__host__ __device__ inline int64_t divide(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0)
    return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Every worker (a warp or a CTA) takes a contiguous run of tiles in the order
// (sequence, key head, block, tile): worker c takes tiles [c * share, (c + 1) *
// share) of the total, so all have the same number whatever the lengths; an
// item cut by a boundary is joined from its pieces afterwards.  A worker
// leaves at most two cut pieces: one that continues an item from the worker
// before, and one whose item goes on in the next.
//
// An item counts as its tiles and, before them, `setup` tiles without keys: what
// fetching its queries and writing its rows costs.  Short items then weigh what
// they take, and a worker whose run ends among an item's setup leaves it whole
// to the next.
__host__ __device__ inline int64_t share_of(int64_t total, int workers, int least) {
  const int64_t share = divide(total + workers - 1, workers);
  return share < least ? least : share;
}

struct Piece {
  int s, h, block;  // item
  int tile, n;      // tiles of it: [tile, tile + n) counted from the item's first
  int whole;        // 1: all of the item's tiles
  int begins;       // 1: starts at the item's first tile
  int ends;         // 1: reaches the item's last tile
};

struct Walker {
  int64_t left;     // tiles still to take
  int s, h, block, tile;
  Seq seq;

  // Positioned at tile `offset` of sequence s0's work (offset below it).
  __host__ __device__ void start(const Batch& b, const Split& w, int s0, int64_t offset,
                                 int64_t count) {
    left = count;
    s = s0;
    seq = load_seq(b, s);
    const int64_t per_head = head_work(w, seq);
    h = static_cast<int>(divide(offset, per_head));
    int64_t rem = offset - h * per_head;
    block = 0;
    for (;;) {
      const int n = block_range(w, seq, block).n + w.setup;
      if (rem < n) break;
      rem -= n;
      ++block;
    }
    tile = static_cast<int>(rem);
  }

  // The next piece; false when the run is done.
  __host__ __device__ bool next(const Batch& b, const Split& w, Piece& p, Range& r) {
    // at least one tile beyond the setup: what remains is a piece
    if (left <= 0 || (tile < w.setup && left <= w.setup - tile)) return false;
    if (block >= row_blocks(w, seq)) {
      block = 0;
      if (++h >= w.hkv) {
        h = 0;
        do {
          if (++s >= b.s) return false;
          seq = load_seq(b, s);
        } while (row_blocks(w, seq) == 0);
      }
    }
    r = block_range(w, seq, block);
    if (tile < w.setup) {
      left -= w.setup - tile;
      tile = w.setup;
    }
    p.s = s;
    p.h = h;
    p.block = block;
    p.tile = tile - w.setup;
    const int rest = r.n - p.tile;
    p.n = left < rest ? static_cast<int>(left) : rest;
    p.begins = p.tile == 0;
    p.ends = p.n == rest;
    p.whole = p.begins && p.ends;
    left -= p.n;
    tile = 0;
    ++block;
    return true;
  }
};

}  // namespace paged
}  // namespace moss
