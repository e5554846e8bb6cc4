// Rotary embedding of queries and keys with an optional RMS norm of every
// head in the same pass (sm_100a), into new tensors (moss_qk_norm_rope) or,
// for a ragged batch of new tokens, with the keys and the values written
// into the pages of a shared history (moss_rope_paged_kv).
//
//   y = x * rsqrt(mean(x^2) + eps) * w     (per head of d, where w is given)
//   (a, b) -> (a cos - b sin, a sin + b cos) for every pair j of the head,
//     angle = position * period^(-2 j / d)
// pairs (2j, 2j + 1) interleaved, or (j, j + d / 2).  Float32 arithmetic, one
// rounding to the output's type.  The angle is formed as a number of turns
// in float64 and reduced there (position * turns_j minus its nearest
// integer), so that a position of millions loses nothing; sine and cosine
// are float32 of the reduced turn.
//
// Bytes bound it: every value is read once and written once.  A row (one
// head of one token) belongs to d / 16 lanes with two 16-byte chunks of 8
// values each, at 8 l and d / 2 + 8 l: both pairings find their partner in
// the same thread, and the norm is a butterfly over d / 16 lanes.  A warp works
// for one token at a time: it forms the token's d / 2 angles (and, paged, finds
// its sequence, position and page) once, keeps their cosines and sines in
// shared memory, and runs over the token's heads, 512 / d rows a step, a batch of
// steps loaded at once.  With few tokens a
// token's steps are spread over several warps, which form the angles again:
// that is cheaper than to wait for one.
#include "paged.cuh"

namespace moss {
namespace qkn {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 256;

struct Args {
  const void* q;
  const void* k;
  const void* v;          // paged only
  const float* q_weight;  // [d] or null
  const float* k_weight;
  void* oq;
  void* ok;               // dense: contiguous [b, hk, t, d]
  uint16_t* k_pages;      // paged: [pages, hk, page_size, d] bf16
  uint16_t* v_pages;
  const void* offset;     // dense: [b] int64 or int32
  paged::Batch batch;     // paged
  int64_t q_stride[3];    // elements: batch, head, token (paged: -, head, token)
  int64_t k_stride[3];
  int64_t v_stride[3];
  float eps;
  int offset_dtype;
  int hq, hk, hv;         // hv: value rows per token (paged: hk, dense: 0)
  int t;                  // dense: tokens per batch entry
  int64_t tokens;         // all of them
  int64_t whole;          // tokens that a warp takes whole; the rest
  int parts;              // are spread over this many warps each
  double turns[kMaxDim / 2];  // period^(-2 j / d) / (2 pi)
};

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&f)[8]) {
  if constexpr (DT == MOSS_BF16) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = pack_bf16x8(f);
  } else {
    float4* s = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    s[0] = make_float4(f[0], f[1], f[2], f[3]);
    s[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// Sequence that owns packed row `row` (whole warp): the number of entries
// q_start[1 ..] at or below it, found by 32-way search.
__device__ __forceinline__ int find_seq(const int64_t* q_start, int s, int64_t row, int lane) {
  int lo = 0, hi = s;  // the answer is in [lo, hi]; entry i stands for q_start[i + 1]
  while (hi > lo) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + (lane + 1) * step - 1;
    const bool below = i < hi && q_start[i + 1] <= row;
    const int m = __popc(__ballot_sync(0xffffffffu, below));
    lo += m * step;
    const int end = lo + step - 1;
    if (end < hi) hi = end;
    if (lo > hi) lo = hi;
  }
  return lo;
}

// A row's two chunks as they were loaded.
template <int DT>
struct Raw {
  uint4 v[DT == MOSS_BF16 ? 2 : 4];
  __device__ __forceinline__ void load(const char* p, int half) {
    constexpr int kPer = DT == MOSS_BF16 ? 1 : 2;  // 16-byte words of 8 values
    const uint4* a = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = a[i];
      v[kPer + i] = a[half / 8 * kPer + i];
    }
  }
  __device__ __forceinline__ void unpack(float (&x)[8], float (&y)[8]) const {
    if constexpr (DT == MOSS_BF16) {
      unpack_bf16x8(v[0], x);
      unpack_bf16x8(v[1], y);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(v[i].x);
        x[4 * i + 1] = __uint_as_float(v[i].y);
        x[4 * i + 2] = __uint_as_float(v[i].z);
        x[4 * i + 3] = __uint_as_float(v[i].w);
        y[4 * i] = __uint_as_float(v[2 + i].x);
        y[4 * i + 1] = __uint_as_float(v[2 + i].y);
        y[4 * i + 2] = __uint_as_float(v[2 + i].z);
        y[4 * i + 3] = __uint_as_float(v[2 + i].w);
      }
    }
  }
};

__device__ __forceinline__ void rotate(float& x, float& y, float c, float s) {
  const float x0 = x, y0 = y;
  x = x0 * c - y0 * s;
  y = x0 * s + y0 * c;
}

__device__ __forceinline__ void scale4(float* x, float r, const float4& w) {
  x[0] *= r * w.x;
  x[1] *= r * w.y;
  x[2] *= r * w.z;
  x[3] *= r * w.w;
}

// Rows of a lane loaded at once, and CTAs per SM: bytes in flight against warps
// that hide one another's angles.  bf16, heads of 128: 16381 tokens x 40 heads,
// four rows and 4 CTAs 60.6 us (5530 GB/s), three and 5 62.5, two and 6 62.4; the
// paged form, which holds more addresses: 10297 tokens x 48 heads, two and 6
// 46.2 (5480 GB/s), two and 5 48.9, three and 4 52.7, one and 8 49.2.  float32
// paged: two and 5 62.1, two and 6 65.6 (registers spilled), one and 6 63.9.
template <int DT, bool PAGED>
constexpr int kBatchRows = DT == MOSS_BF16 && !PAGED ? 4 : 2;
template <int DT, bool PAGED>
constexpr int kResident = !PAGED ? 4 : (DT == MOSS_BF16 ? 6 : 5);

template <int DT, int D, bool PAGED, bool PAIRS>
__global__ void __launch_bounds__(kThreads, kResident<DT, PAGED>)
    norm_rope_kernel(const __grid_constant__ Args a) {
  constexpr int L = D / 16;       // lanes per row
  constexpr int kRows = 32 / L;   // rows per step
  constexpr int kIn = DT == MOSS_BF16 ? 2 : 4, kOut = PAGED ? 2 : kIn;  // bytes of a value
  constexpr int kBatch = kBatchRows<DT, PAGED>;
  // A lane's 8 angles and 16 weights as four 16-byte words each, the same word
  // of a row's lanes side by side: lane after lane they shared banks, and took
  // 65 us where this takes 62 (paged: 58, 50).
  __shared__ float4 cs_smem[kWarps][4 * L];
  __shared__ float4 weights[2][4 * L];
  __shared__ double turns[D / 2];
  for (int i = threadIdx.x; i < D; i += kThreads) {
    const int at = (((i / (D / 2) * 2 + i % 8 / 4) * L + i % (D / 2) / 8) << 2) + i % 4;
    if (a.q_weight != nullptr) reinterpret_cast<float*>(weights[0])[at] = a.q_weight[i];
    if (a.k_weight != nullptr) reinterpret_cast<float*>(weights[1])[at] = a.k_weight[i];
  }
  for (int i = threadIdx.x; i < D / 2; i += kThreads) turns[i] = a.turns[i];
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane % L, place = lane / L;
  float4* cs = cs_smem[warp];
  // of angle j: the word's place in pairs of floats
  auto angle_at = [](int j) {
    const int word = PAIRS ? j / (D / 4) * 2 + j % 4 / 2 : j % 8 / 2;
    const int owner = PAIRS ? j % (D / 4) / 4 : j / 8;
    return (word * L + owner) * 2 + j % 2;
  };
  const int steps_q = (a.hq + kRows - 1) / kRows, steps_k = (a.hk + kRows - 1) / kRows;
  const int steps = steps_q + steps_k + (a.hv + kRows - 1) / kRows;
  const int64_t units = a.whole + (a.tokens - a.whole) * a.parts;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp; unit < units;
       unit += static_cast<int64_t>(gridDim.x) * kWarps) {
    int64_t token = unit;
    int begin = 0, end = steps;
    if (unit >= a.whole) {
      const int64_t rest = paged::divide(unit - a.whole, a.parts);
      const int part = static_cast<int>(unit - a.whole - rest * a.parts);
      token = a.whole + rest;
      begin = steps * part / a.parts;
      end = steps * (part + 1) / a.parts;
    }
    int64_t batch = 0, step_at = token, page_at = -1, pos;
    bool owned = true;
    if constexpr (PAGED) {
      const paged::Batch& b = a.batch;
      const int s = find_seq(b.q_start, b.s, token, lane);
      pos = 0;
      owned = s < b.s && token >= b.q_start[0];
      if (owned) {
        pos = b.kv_len[s] - (b.q_start[s + 1] - token);
        const int64_t slot = pos >> b.page_shift;
        int page = -1;
        if (pos >= 0 && slot < b.max_pages)
          page = b.table[static_cast<int64_t>(s) * b.max_pages + slot];
        if (page >= 0 && page < b.pages)
          page_at = ((static_cast<int64_t>(page) * a.hk) << b.page_shift) +
                    (pos & ((1 << b.page_shift) - 1));
        else if (lane == 0)
          record_device_error(MOSS_ERR_VALUE);
      }
    } else {
      batch = paged::divide(token, a.t);
      step_at = token - batch * a.t;
      pos = step_at + (a.offset_dtype == 0
                           ? static_cast<const int64_t*>(a.offset)[batch]
                           : static_cast<int64_t>(static_cast<const int32_t*>(a.offset)[batch]));
    }
    if (!owned) continue;  // a row of no sequence
#pragma unroll
    for (int j = lane; j < D / 2; j += 32) {
      const double x = static_cast<double>(pos) * turns[j];
      float sn, c;
      sincospif(static_cast<float>(2.0 * (x - rint(x))), &sn, &c);
      reinterpret_cast<float2*>(cs)[angle_at(j)] = make_float2(c, sn);
    }
    __syncwarp();

#pragma unroll 1
    for (int kind = 0; kind < (PAGED ? 3 : 2); ++kind) {
      const int before = kind == 0 ? 0 : (kind == 1 ? steps_q : steps_q + steps_k);
      const int heads = kind == 0 ? a.hq : (kind == 1 ? a.hk : a.hv);
      const int first = begin > before ? begin - before : 0;
      const int all = (heads + kRows - 1) / kRows;
      const int last = end - before < all ? end - before : all;
      if (first >= last) continue;
      if (PAGED && kind > 0 && page_at < 0) continue;  // nowhere to store
      int head = first * kRows + place;
      const int64_t* st = kind == 0 ? a.q_stride : (kind == 1 ? a.k_stride : a.v_stride);
      // byte addresses of this lane's first chunk, where it comes from and goes
      const char* src = static_cast<const char*>(kind == 0 ? a.q : (kind == 1 ? a.k : a.v)) +
                        (batch * st[0] + step_at * st[2] + head * st[1] + sub * 8) * kIn;
      const int64_t src_step = kRows * st[1] * kIn;
      char* dst;
      int64_t dst_step;
      if constexpr (PAGED) {
        dst_step = kind == 0 ? D : static_cast<int64_t>(D) << a.batch.page_shift;
        dst = kind == 0 ? static_cast<char*>(a.oq) + token * a.hq * D * kOut
                        : reinterpret_cast<char*>(kind == 1 ? a.k_pages : a.v_pages) +
                              page_at * D * kOut;
      } else {
        dst_step = static_cast<int64_t>(a.t) * D;
        dst = static_cast<char*>(kind == 0 ? a.oq : a.ok) +
              (batch * heads * a.t + step_at) * D * kOut;
      }
      dst += (head * dst_step + sub * 8) * kOut;
      dst_step *= kRows * kOut;
      const bool normed = kind == 0 ? a.q_weight != nullptr : kind == 1 && a.k_weight != nullptr;
      const float4* weight = weights[kind & 1] + sub;
#pragma unroll 1
      for (int i0 = first; i0 < last; i0 += kBatch) {
        // a batch's loads all in flight before the first is used
        Raw<DT> raw[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
          if (i0 + b < last && head + b * kRows < heads) raw[b].load(src + b * src_step, D / 2);
        src += kBatch * src_step;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (i0 + b >= last) break;
          const bool on = head < heads;  // the butterfly is warp-wide
          float x[8], y[8];
          raw[b].unpack(x, y);
          head += kRows;
          if (normed) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += x[e] * x[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += y[e] * y[e];
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float r = rsqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
              scale4(x + e, r, weight[e / 4 * L]);
              scale4(y + e, r, weight[(2 + e / 4) * L]);
            }
          }
          if (kind < 2) {
            if constexpr (PAIRS) {
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const float4 ca = cs[e / 2 * L + sub];
                rotate(x[2 * e], x[2 * e + 1], ca.x, ca.y);
                rotate(x[2 * e + 2], x[2 * e + 3], ca.z, ca.w);
                const float4 cb = cs[(2 + e / 2) * L + sub];
                rotate(y[2 * e], y[2 * e + 1], cb.x, cb.y);
                rotate(y[2 * e + 2], y[2 * e + 3], cb.z, cb.w);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                const float4 c = cs[e / 2 * L + sub];
                rotate(x[e], y[e], c.x, c.y);
                rotate(x[e + 1], y[e + 1], c.z, c.w);
              }
            }
          }
          if (on) {
            // the pages and the queries for them are bf16, what the attention reads
            store8<PAGED ? MOSS_BF16 : DT>(dst, 0, x);
            store8<PAGED ? MOSS_BF16 : DT>(dst, D / 2, y);
          }
          dst += dst_step;
        }
      }
    }
    __syncwarp();  // the angles may be written again
  }
  // rows beyond the packed ones, whose keys are missing (nobody waits for this load)
  if constexpr (PAGED) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.batch.q_start[a.batch.s] > a.batch.n)
      record_device_error(MOSS_ERR_VALUE);
  }
}

template <int DT, int D, bool PAGED, bool PAIRS>
int launch(Args& a, cudaStream_t stream, const char* name) {
  // Every resident warp takes the same number of whole tokens; the steps of those
  // that remain (of all, where there are few) are spread over as many warps.
  constexpr int kRows = 512 / D;
  auto up = [](int x) { return (x + kRows - 1) / kRows; };
  const int steps = up(a.hq) + up(a.hk) + up(a.hv);
  auto kernel = norm_rope_kernel<DT, D, PAGED, PAIRS>;
  static int64_t resident[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) dev = 0;
  if (resident[dev] == 0) resident[dev] = persistent_grid(kernel, kThreads, 0, INT64_MAX);
  const int64_t warps = resident[dev] * kWarps;
  a.whole = a.tokens / warps * warps;
  const int64_t rest = a.tokens - a.whole;
  const int64_t parts = rest > 0 ? warps / rest : 1;
  a.parts = parts < steps ? static_cast<int>(parts) : steps;
  const int64_t work = (a.whole + rest * a.parts + kWarps - 1) / kWarps;
  const int64_t grid = work < resident[dev] ? work : resident[dev];
  kernel<<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  return launch_status(name);
}

template <int DT, bool PAGED, bool PAIRS>
int by_dim(Args& a, int64_t d, cudaStream_t stream, const char* name) {
  switch (d) {
    case 32:
      if constexpr (!PAGED) return launch<DT, 32, PAGED, PAIRS>(a, stream, name);
      break;
    case 64: return launch<DT, 64, PAGED, PAIRS>(a, stream, name);
    case 128: return launch<DT, 128, PAGED, PAIRS>(a, stream, name);
    case 256:
      if constexpr (!PAGED) return launch<DT, 256, PAGED, PAIRS>(a, stream, name);
      break;
  }
  return fail(MOSS_ERR_UNSUPPORTED, "%s: unsupported head width", name);
}

template <bool PAGED>
int dispatch(Args& a, int dtype, int64_t d, int interleaved, cudaStream_t stream,
             const char* name) {
  if (dtype == MOSS_BF16)
    return interleaved ? by_dim<MOSS_BF16, PAGED, true>(a, d, stream, name)
                       : by_dim<MOSS_BF16, PAGED, false>(a, d, stream, name);
  return interleaved ? by_dim<MOSS_F32, PAGED, true>(a, d, stream, name)
                     : by_dim<MOSS_F32, PAGED, false>(a, d, stream, name);
}

// period^(-2 j / d) / (2 pi) in float64: exponentials of the coarse and the
// fine part of j, multiplied (two roundings, about 2^-52 relative).
void fill_turns(double* turns, int64_t d, double period) {
  const double c = -2.0 * log(period) / static_cast<double>(d);
  double fine[16];
  const int half = static_cast<int>(d / 2);
  for (int j = 0; j < 16; ++j) fine[j] = exp(c * j) * 0.15915494309189533577;
  for (int j0 = 0; j0 < half; j0 += 16) {
    const double coarse = exp(c * j0);
    for (int j = 0; j < 16; ++j) turns[j0 + j] = coarse * fine[j];
  }
}

// Rows are read as 16-byte chunks.
bool chunked(const void* p, int dtype, const int64_t* strides, int n) {
  const int per = dtype == MOSS_BF16 ? 8 : 4;
  if (!aligned16(p)) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] % per) return false;
  return true;
}

}  // namespace qkn
}  // namespace moss

using namespace moss;

extern "C" int moss_qk_norm_rope(const void* q, const void* k, int dtype, const float* q_weight,
                                 const float* k_weight, float eps, const void* offset,
                                 int offset_dtype, double max_period, int interleaved, void* oq,
                                 void* ok, int64_t b, int64_t hq, int64_t hk, int64_t t, int64_t d,
                                 const int64_t* q_strides, const int64_t* k_strides,
                                 void* stream) {
  const char* name = "moss_qk_norm_rope";
  if (b < 0 || hq < 1 || hk < 1 || t < 0 || d < 2 || d % 2)
    return fail(MOSS_ERR_VALUE, "%s: bad shape", name);
  if (dtype != MOSS_F32 && dtype != MOSS_BF16)
    return fail(MOSS_ERR_VALUE, "%s: unknown dtype %d", name, dtype);
  if (offset_dtype != 0 && offset_dtype != 1)
    return fail(MOSS_ERR_VALUE, "%s: offsets must be int64 or int32", name);
  if (!(max_period > 0.0) || !isfinite(max_period))
    return fail(MOSS_ERR_VALUE, "%s: max_period must be positive and finite", name);
  if (!(eps >= 0.0f)) return fail(MOSS_ERR_VALUE, "%s: eps must not be negative", name);
  if (d != 32 && d != 64 && d != 128 && d != 256)
    return fail(MOSS_ERR_UNSUPPORTED, "%s: heads of 32, 64, 128 or 256", name);
  if (b == 0 || t == 0) return MOSS_OK;
  if (!q || !k || !offset || !oq || !ok || !q_strides || !k_strides)
    return fail(MOSS_ERR_VALUE, "%s: null pointer", name);
  if (hq + hk > (1 << 16) || t > 0x7fffffff || b > (1LL << 40) / t)
    return fail(MOSS_ERR_UNSUPPORTED, "%s: too large", name);
  if (q_strides[3] != 1 || k_strides[3] != 1 || !qkn::chunked(q, dtype, q_strides, 3) ||
      !qkn::chunked(k, dtype, k_strides, 3) || !aligned16(oq) || !aligned16(ok) ||
      (q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight)))
    return fail(MOSS_ERR_UNSUPPORTED, "%s: rows must be contiguous and 16-byte aligned", name);
  qkn::Args a{};
  a.q = q;
  a.k = k;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.oq = oq;
  a.ok = ok;
  a.offset = offset;
  a.offset_dtype = offset_dtype;
  a.eps = eps;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = q_strides[i];
    a.k_stride[i] = k_strides[i];
  }
  a.hq = static_cast<int>(hq);
  a.hk = static_cast<int>(hk);
  a.hv = 0;
  a.t = static_cast<int>(t);
  a.tokens = b * t;
  qkn::fill_turns(a.turns, d, max_period);
  return qkn::dispatch<false>(a, dtype, d, interleaved, as_stream(stream), name);
}

extern "C" int moss_rope_paged_kv(const void* q, const void* k, const void* v, int dtype,
                                  const float* q_weight, const float* k_weight, float eps,
                                  const int64_t* q_start, const int64_t* kv_len,
                                  const int32_t* page_table, double max_period, int interleaved,
                                  void* oq, void* k_pages, void* v_pages, int64_t n, int64_t s,
                                  int64_t hq, int64_t hkv, int64_t d, int64_t pages,
                                  int64_t page_size, int64_t max_pages, const int64_t* q_strides,
                                  const int64_t* k_strides, const int64_t* v_strides,
                                  void* stream) {
  const char* name = "moss_rope_paged_kv";
  if (n < 0 || s < 0 || hq < 1 || hkv < 1 || d < 2 || pages < 0 || max_pages < 0)
    return fail(MOSS_ERR_VALUE, "%s: bad shape", name);
  if (dtype != MOSS_F32 && dtype != MOSS_BF16)
    return fail(MOSS_ERR_VALUE, "%s: unknown dtype %d", name, dtype);
  if (!(max_period > 0.0) || !isfinite(max_period))
    return fail(MOSS_ERR_VALUE, "%s: max_period must be positive and finite", name);
  if (!(eps >= 0.0f)) return fail(MOSS_ERR_VALUE, "%s: eps must not be negative", name);
  if (d != 64 && d != 128) return fail(MOSS_ERR_UNSUPPORTED, "%s: heads of 64 or 128", name);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return fail(MOSS_ERR_UNSUPPORTED, "%s: pages of 16, 32, 64, 128 or 256 positions", name);
  if (n == 0 || s == 0) return MOSS_OK;
  if (!q || !k || !v || !q_start || !kv_len || !page_table || !oq || !k_pages || !v_pages ||
      !q_strides || !k_strides || !v_strides)
    return fail(MOSS_ERR_VALUE, "%s: null pointer", name);
  if (hq + 2 * hkv > (1 << 16) || n > 0x3fffffff || s > 0x3fffffff || pages > 0x7fffffff ||
      max_pages > 0x7fffffff / page_size)
    return fail(MOSS_ERR_UNSUPPORTED, "%s: too large", name);
  if (q_strides[2] != 1 || k_strides[2] != 1 || v_strides[2] != 1 ||
      !qkn::chunked(q, dtype, q_strides, 2) || !qkn::chunked(k, dtype, k_strides, 2) ||
      !qkn::chunked(v, dtype, v_strides, 2) || !aligned16(oq) || !aligned16(k_pages) ||
      !aligned16(v_pages) || (q_weight && !aligned16(q_weight)) ||
      (k_weight && !aligned16(k_weight)))
    return fail(MOSS_ERR_UNSUPPORTED, "%s: rows must be contiguous and 16-byte aligned", name);
  qkn::Args a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.oq = oq;
  a.k_pages = static_cast<uint16_t*>(k_pages);
  a.v_pages = static_cast<uint16_t*>(v_pages);
  a.eps = eps;
  a.batch.q_start = q_start;
  a.batch.kv_len = kv_len;
  a.batch.table = page_table;
  a.batch.n = static_cast<int>(n);
  a.batch.s = static_cast<int>(s);
  a.batch.max_pages = static_cast<int>(max_pages);
  a.batch.pages = static_cast<int>(pages);
  while ((1 << a.batch.page_shift) < page_size) ++a.batch.page_shift;
  a.q_stride[1] = q_strides[1];
  a.q_stride[2] = q_strides[0];
  a.k_stride[1] = k_strides[1];
  a.k_stride[2] = k_strides[0];
  a.v_stride[1] = v_strides[1];
  a.v_stride[2] = v_strides[0];
  a.hq = static_cast<int>(hq);
  a.hk = static_cast<int>(hkv);
  a.hv = static_cast<int>(hkv);
  a.tokens = n;
  qkn::fill_turns(a.turns, d, max_period);
  return qkn::dispatch<true>(a, dtype, d, interleaved, as_stream(stream), name);
}
