// Group norm of the rows of ragged samples (channels last) with the gated activation behind it, and its gradients.
//
// A group is a range of channels, the copies of fields of one order; its statistics run over the rows of a sample and the
// copies.  Scalars: mu = mean, v = mean (x - mu)^2.  Fields of order l > 0: mu = 0, v = mean |x|^2, which commutes with
// rotations.  With r = (v + eps)^-1/2: z = (x - mu) r w + b; the activation follows.  Backward, with a = dz w, xhat = (x - mu) r and M =
// rows * copies: dx = r (a - [scalars] sum(a) / M - xhat sum(a xhat) / M), dw = sum dz xhat, db = sum dz.
//
// Memory-bound: each direction is two passes over the rows, sums first.  The rows are cut into equal ranges, one to a block, two blocks to an SM,
// whatever the samples' lengths; a block walks through the pieces of samples in its range and leaves a partial result for each, and the second
// pass adds up those of a sample in a fixed order (no atomics: the same bits every time).  Rows come by bulk copies into a ring of
// tiles: with loads in the threads themselves, registers for the rows in flight left room for two blocks of
// 256 threads, which waited for memory half of the time.
//
// 786432 rows of 128 in bf16: sums 53 us (3.8 TB/s), second pass 84 (4.8 TB/s read and written).  65536 rows of 256 in float32, all in L2: 22 and 23, backward 41 and
// 42.  A launch on next to nothing takes 6 to 8 us (tables, offsets, the copies' first latency, sums at the end); from there on instructions bound it, 10 to 30 a value
// at half of the issue slots: more warps, bigger tiles, and a second pass from the end (to find rows in L2) changed nothing or cost elsewhere.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ssc_common.cuh"
#include "ssc_rows_act.cuh"
#include "ssc_tc_ptx.cuh"

namespace ssc {
namespace {

struct GnTable {
  const int32_t *group_of_channel, *field_of_channel, *scalar_of_channel;   // [c]
  const int32_t *gate_of_channel;                                           // [c_out]: -2 copy, -1 scalar activation, else the gate
  const int32_t *field_first, *field_len, *field_scalar;                    // [n_field]
  const int32_t *gate_field;                                                // [n_gate]
  const int32_t *group_first, *group_len, *group_copies;                    // [n_group]
};
struct GnArgs {
  const void *x, *gy;
  void *out;
  int n, c, c_out, n_gate, n_group, n_field, n_scalar, batch;
  const int32_t *offsets;
  GnTable t;
  const float *weight, *bias;
  float eps;
  int scalar_act, gate_act;
  int threads, tile, range, blocks, stages;    // threads and rows of a tile and of a block; blocks; tiles of the ring
  uint32_t x_bytes, stage_bytes;               // of a stage: rows of x, then of gy
  float *partial;      // [blocks + batch][n_group][2]: block b's piece of sample s at b + s
  float *fields;       // [blocks][n_field + n_scalar]
  float *stats;        // [batch][n_group][2]: mu, r
  float *d_weight, *d_bias;
  int32_t *status, *alarm;
};

constexpr int kGnThreads = 512;             // at most; 256 where a row has fewer slots than that
constexpr int kGnStages = 8;
constexpr int kGnGateRows = 4;             // rows side by side in the gates' part of the backward passes, where a row leaves room for fewer
constexpr int kGnSum = 32;                  // columns of d_weight | d_bias to a block of the second backward pass

// Rows of T, VEC channels to a thread.  WHOLE: the channels are a multiple of VEC, so that rows start at multiples of VEC; else the last thread of
// a row has fewer (`many`), and values are read and written one by one.  (A channel to a thread where they are no multiple took three times as long:
// forward and backward of 171981 rows of 135 channels in fp32 617 us.)
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };
template <class T, int VEC, bool WHOLE>
__device__ __forceinline__ void load(const T *p, float *v, int many) {
  if (WHOLE) {
    const Pack<T, VEC> k = *(const Pack<T, VEC> *)p;
#pragma unroll
    for (int q = 0; q < VEC; ++q) v[q] = (float)k.v[q];
  } else {
#pragma unroll
    for (int q = 0; q < VEC; ++q) v[q] = q < many ? (float)p[q] : 0.f;
  }
}
template <class T, int VEC, bool WHOLE>
__device__ __forceinline__ void store(T *p, const float *v, int many) {
  if (WHOLE) {
    Pack<T, VEC> k;
#pragma unroll
    for (int q = 0; q < VEC; ++q) k.v[q] = (T)v[q];
    *(Pack<T, VEC> *)p = k;
  } else {
#pragma unroll
    for (int q = 0; q < VEC; ++q)
      if (q < many) p[q] = (T)v[q];
  }
}

// The block's range of rows as tiles of a ring in shared memory, which thread 0 feeds as it goes: one tile behind, so that it does not wait for
// the slowest warp.  (A ninth warp that feeds it costs a quarter of the registers.)
struct GnRing {
  uint32_t ring, full, empty;
  char *base;
  volatile int *abort_flag;
  int r0, r1, x_row, gy_row;
  int issued;               // thread 0: tiles so far, the slot of the next one and the phase of its copies
  uint32_t put_slot, put_phase;
  // the tile they are at, its first row, its slot and the slot's phase, whether it has been waited for
  int first;
  uint32_t slot, phase;
  bool here;

  __device__ __forceinline__ void open(const GnArgs &a, int block, char *smem, uint64_t *bars, volatile int *flag, int size, int size_gy) {
    ring = smem_u32(smem);
    base = smem;
    full = smem_u32(bars);
    empty = full + 8 * kGnStages;
    abort_flag = flag;
    r0 = (int)min((long long)block * a.range, (long long)a.n);
    r1 = (int)min((long long)r0 + a.range, (long long)a.n);
    first = r0;
    slot = phase = 0;
    here = false;
    x_row = a.c * size;
    gy_row = a.c_out * size_gy;
    issued = 0;
    put_slot = put_phase = 0;
    if (threadIdx.x == 0) {
      for (int s = 0; s < a.stages; ++s) {
        mbar_init(full + 8 * s, 1);
        mbar_init(empty + 8 * s, a.threads / 32);
      }
      *flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int s = 0; s < a.stages; ++s) issue(a);
  }
  // (one thread) rows [row, row + rows) of a matrix of `bytes` wide rows; returns what the copy engine brings, which takes 16 bytes at a time:
  // the end of the last row of all may be left to this thread.
  static __device__ __forceinline__ uint32_t piece(const void *src, int row, int rows, int bytes, bool issue, char *dst, uint32_t at, uint32_t bar) {
    const char *from = (const char *)src + (size_t)row * bytes;
    const uint32_t all = (uint32_t)rows * bytes, whole = all & ~15u;
    if (!issue) {
      for (uint32_t i = whole; i < all; i += 2) *(uint16_t *)(dst + i) = *(const uint16_t *)(from + i);
    } else if (whole) {
      bulk_g2s(at, from, whole, bar);
    }
    return whole;
  }
  // (thread 0) the next tile into its slot, once all warps have left the one that was there.
  __device__ __forceinline__ void issue(const GnArgs &a) {
    const int row = r0 + issued * a.tile;
    if (row >= r1) return;
    const uint32_t at = put_slot * a.stage_bytes, bar = full + 8 * put_slot;
    if (issued >= a.stages && !mbar_wait(empty + 8 * put_slot, put_phase ^ 1, abort_flag)) return;
    const int rows = min(a.tile, r1 - row);
    uint32_t bytes = piece(a.x, row, rows, x_row, false, base + at, 0, 0);
    if (gy_row) bytes += piece(a.gy, row, rows, gy_row, false, base + at + a.x_bytes, 0, 0);
    mbar_expect_tx(bar, bytes);
    piece(a.x, row, rows, x_row, true, nullptr, ring + at, bar);
    if (gy_row) piece(a.gy, row, rows, gy_row, true, nullptr, ring + at + a.x_bytes, bar);
    ++issued;
    if (++put_slot == (uint32_t)a.stages) put_slot = 0, put_phase ^= 1;
  }
  // The block's end: copies that nobody has waited for arrive before it leaves.
  __device__ __forceinline__ void close(const GnArgs &a) {
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0) {
      for (int s = max(issued - a.stages, 0); s < issued; ++s) mbar_wait_drain(full + 8 * (s % a.stages), (s / a.stages) & 1);
      report_expired(a.status, a.alarm);
    }
  }
  // The tile at hand.  After a wait that has run out the walk goes on to its end, on whatever is there: the consumers wait for one
  // another on the way.
  __device__ __forceinline__ const char *tile(const GnArgs &a) {
    if (!here) {
      (void)mbar_wait(full + 8 * slot, phase, abort_flag);
      here = true;
    }
    return base + slot * a.stage_bytes;
  }
  __device__ __forceinline__ int end(const GnArgs &a) const { return min(first + a.tile, r1); }
  // Rows up to `row` are done.
  __device__ __forceinline__ void release(const GnArgs &a, int row) {
    if (row < end(a)) return;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(empty + 8 * slot);
    if (threadIdx.x == 0 && first > r0) issue(a);
    first += a.tile;
    here = false;
    if (++slot == (uint32_t)a.stages) slot = 0, phase ^= 1;
  }
};

// The sample that holds a row (-1 before the first one, batch behind the last one), by 32 looks at a time; and where its piece ends.  Offsets are
// cut down to the rows; in a list that does not ascend the pieces are arbitrary, but the walk still ends.
struct GnWalk {
  int s, lo, hi;
  __device__ __forceinline__ int edge(const GnArgs &a, int i) const { return min(max(a.offsets[i], 0), a.n); }
  __device__ __forceinline__ void find(const GnArgs &a, int row) {
    const int lane = threadIdx.x & 31;
    int from = 0, to = a.batch + 1;           // offsets that are at most row: their number lies between
    while (from < to) {
      const int step = (to - from + 31) / 32, at = from + (lane + 1) * step - 1;
      const int many = __popc(__ballot_sync(0xffffffffu, at < to && a.offsets[at] <= row));
      from += many * step;
      to = min(to, from + step - 1);
    }
    s = from - 1;
    place(a, row);
  }
  __device__ __forceinline__ void place(const GnArgs &a, int row) {
    for (;; ++s) {
      lo = s < 0 ? 0 : edge(a, s);
      hi = s >= a.batch ? a.n : edge(a, s + 1);
      if (s >= a.batch || hi > row) break;
    }
  }
  __device__ __forceinline__ bool live(const GnArgs &a) const { return s >= 0 && s < a.batch; }
};

// First pass, forward: mean and sum of squared distances of each group of a piece.  A thread takes four rows at a time, exactly
// (mean first), and adds them to its running values (Chan et al. 1979): sums of squares and of values alone would lose the
// variance of rows far from zero.
template <class T, int VEC, bool WHOLE>
__global__ void __launch_bounds__(kGnThreads, 1) gn_stats_kernel(GnArgs a) {
  after_previous();
  extern __shared__ __align__(128) char smem[];
  __shared__ alignas(8) uint64_t bars[2 * kGnStages];
  __shared__ volatile int abort_flag;
  GnRing ring;
  ring.open(a, blockIdx.x, smem, bars, &abort_flag, sizeof(T), 0);
  const int t = threadIdx.x;
  float *sm = (float *)(smem + a.stages * a.stage_bytes);       // [R][c] means, [R][c] squares
  const int slots = (a.c + VEC - 1) / VEC, R = a.threads / slots, ty = t / slots, ch = (t - ty * slots) * VEC, many = min(VEC, a.c - ch);
  const bool works = ty < R;
  float *sq_s = sm + R * a.c, *sums = sq_s + R * a.c, centred[VEC], quarter[VEC];       // sums: [c] twice
#pragma unroll
  for (int q = 0; q < VEC; ++q) centred[q] = works && q < many && a.t.scalar_of_channel[ch + q] >= 0 ? 1.f : 0.f, quarter[q] = 0.25f * centred[q];
  // (what the ends of pieces look up first comes with the first rows)
  const int lane = t & 31, first_group = t >> 5;
  int my_from = 0, my_len = 0, shift = 0;
  while (shift < 5 && a.c << (shift + 1) <= a.threads) ++shift;        // lanes to a channel at the end of a piece
  const int part = t & ((1 << shift) - 1);
  if (first_group < a.n_group) my_from = a.t.group_first[first_group], my_len = a.t.group_len[first_group];
  GnWalk walk;
  if (ring.r0 < ring.r1) walk.find(a, ring.r0);
  for (int row = ring.r0; row < ring.r1;) {
    const int begin = row, end = min(walk.hi, ring.r1);
    float mean[VEC] = {}, sq[VEC] = {}, have = 0.f;
    while (row < end) {
      const T *x = (const T *)ring.tile(a) + ch;
      const int first = ring.first, last = min(end, ring.end(a));
      if (works && walk.live(a)) {
        int i = row - first + ty;
        const int stop = last - first;
        for (; i + 3 * R < stop; i += 4 * R) {
          float v[4][VEC];
#pragma unroll
          for (int u = 0; u < 4; ++u) load<T, VEC, WHOLE>(x + (i + u * R) * a.c, v[u], many);
          const float f = __fdividef(4.f, have + 4.f);
          float mb[VEC], d[VEC], s[VEC];
          multiply_add<VEC>(mb, v[0], 1.f, v[1]);
          multiply_add<VEC>(d, v[2], 1.f, v[3]);
          multiply_add<VEC>(mb, mb, 1.f, d);
          multiply<VEC>(mb, mb, quarter);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            multiply_add<VEC>(d, mb, -1.f, v[u]);
            if (u == 0) multiply<VEC>(s, d, d);
            else multiply_add<VEC>(s, d, d, s);
          }
          multiply_add<VEC>(d, mean, -1.f, mb);
          multiply_add<VEC>(mean, d, f, mean);
          multiply<VEC>(mb, d, have * f);
          multiply_add<VEC>(s, mb, d, s);
          multiply_add<VEC>(sq, sq, 1.f, s);
          have += 4.f;
        }
        for (; i < stop; i += R) {
          float v[VEC];
          load<T, VEC, WHOLE>(x + i * a.c, v, many);
          const float f = __fdividef(1.f, have + 1.f);
#pragma unroll
          for (int q = 0; q < VEC; ++q) {
            const float mb = v[q] * centred[q], d = mb - mean[q], e = v[q] - mb;
            mean[q] = fmaf(d, f, mean[q]);
            sq[q] += fmaf(have * f * d, d, e * e);
          }
          have += 1.f;
        }
      }
      ring.release(a, last);
      row = last;
    }
    if (walk.live(a)) {
      if (works) {
#pragma unroll
        for (int q = 0; q < VEC; ++q)
          if (q < many) {
            sm[ty * a.c + ch + q] = mean[q];
            sq_s[ty * a.c + ch + q] = sq[q];
          }
      }
      __shared__ float count[kGnThreads];
      if (works && ch == 0) count[ty] = have;
      __syncthreads();
      // the mean of what is put together first, then the squares about it: about a channel, a row or a piece that lies far from the
      // others (a thousand spreads) they would be as many times the variance, 1e-5 of which is lost; and the mean once more, which is
      // off by a rounding of such a one.  (3501 rows of 38 channels in 290 pieces 5.9 us for the pass, 5.7 in one go about a first mean; 786432 rows of
      // 128 in bf16 52.9 and 50.4.)
      const float rows = (float)(end - begin);
      for (int i0 = 0; i0 < a.c; i0 += a.threads >> shift) {
        const int i = i0 + (t >> shift), at = i < a.c ? i : 0;
        const float about = sm[at];
        float u = 0.f, v = 0.f, left = 0.f;
#pragma unroll 2
        for (int r = part; r < R; r += 1 << shift) u = fmaf(count[r], sm[r * a.c + at] - about, u);
        for (int d = 1 << shift >> 1; d > 0; d >>= 1) u += __shfl_xor_sync(0xffffffffu, u, d);
        const float mean = about + __fdividef(u, rows);
#pragma unroll 2
        for (int r = part; r < R; r += 1 << shift) {
          const float d = sm[r * a.c + at] - mean, nd = count[r] * d;
          left += nd;
          v += fmaf(nd, d, sq_s[r * a.c + at]);
        }
        for (int d = 1 << shift >> 1; d > 0; d >>= 1) left += __shfl_xor_sync(0xffffffffu, left, d), v += __shfl_xor_sync(0xffffffffu, v, d);
        if (part == 0 && i < a.c) {
          sums[i] = mean + __fdividef(left, rows);
          sums[a.c + i] = v;
        }
      }
      __syncthreads();
      for (int g = first_group; g < a.n_group; g += a.threads >> 5) {
        const bool mine = g == first_group;
        const int from = mine ? my_from : a.t.group_first[g], len = mine ? my_len : a.t.group_len[g];
        const float about = sums[from];
        float u = 0.f, v = 0.f;
        for (int i = lane; i < len; i += 32) u += sums[from + i] - about;
        for (int d = 16; d > 0; d >>= 1) u += __shfl_xor_sync(0xffffffffu, u, d);
        const float mean = about + __fdividef(u, (float)len);
        float left = 0.f;
        for (int i = lane; i < len; i += 32) {
          const float d = sums[from + i] - mean;
          left += d;
          v += fmaf(rows * d, d, sums[a.c + from + i]);
        }
        for (int d = 16; d > 0; d >>= 1) left += __shfl_xor_sync(0xffffffffu, left, d), v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == 0) *(float2 *)(a.partial + ((size_t)(blockIdx.x + walk.s) * a.n_group + g) * 2) = {mean + __fdividef(left, (float)len), v};
      }
      __syncthreads();
    }
    if (row < ring.r1) walk.place(a, row);
  }
  ring.close(a);
}

// The partial results of the walk's sample: from block `first` on, `many` of them.
__device__ __forceinline__ void sample_pieces(const GnArgs &a, const GnWalk &k, int &first, int &many) {
  first = k.lo / a.range;
  many = k.hi > k.lo ? (k.hi - 1) / a.range - first + 1 : 0;
}
__device__ __forceinline__ int piece_rows(const GnArgs &a, const GnWalk &k, int block) {
  const int lo = block * a.range;          // (a range is a small share of at most 2^30 rows)
  return min(lo + a.range, k.hi) - max(lo, k.lo);
}

// What pieces of a sample are put together from: sums, or rows with their mean and the squares about it (Chan et al. 1979).
struct GnSums {
  float u, v;
  __device__ __forceinline__ void add(const GnSums &o) { u += o.u, v += o.v; }
  __device__ __forceinline__ GnSums across(int d) const { return {__shfl_xor_sync(0xffffffffu, u, d), __shfl_xor_sync(0xffffffffu, v, d)}; }
};
struct GnMoments {
  float rows, mean, sq;
  __device__ __forceinline__ void add(const GnMoments &o) {
    const float both = rows + o.rows, share = both > 0.f ? __fdividef(o.rows, both) : 0.f, d = o.mean - mean;
    sq += fmaf(rows * share * d, d, o.sq);       // (nothing times any d is nothing: d * d may be beyond the range)
    mean = fmaf(d, share, mean);
    rows = both;
  }
  __device__ __forceinline__ GnMoments across(int d) const {
    return {__shfl_xor_sync(0xffffffffu, rows, d), __shfl_xor_sync(0xffffffffu, mean, d), __shfl_xor_sync(0xffffffffu, sq, d)};
  }
};
// V of each group over the partial results of a sample: load(group, piece, its result), end(group, V).
// Few pieces: up to eight lanes to a group.  Many, as in a sample that all blocks share: lanes side by side read neighbouring groups, each warp
// its share of the pieces.  (Two samples of 1750 rows in 290 pieces, 32 groups: a group to a warp, which fetches a sector for each of
// its results, 16.3 us for the second pass forward, this way 11.5; one sample of 203437 rows, 8 groups 17.9 and 16.8.)
constexpr int kGnPieces = 4;               // in flight
template <class V, class Load, class End>
__device__ __forceinline__ void sample_sums(const GnArgs &a, const float *from, int many, Load load, End end) {
  const float2 *all = (const float2 *)from;
  const int lane = threadIdx.x & 31;
  if (many <= 8) {
    const int width = many <= 4 ? 4 : 8, at = lane & (width - 1);
    for (int g0 = 0; g0 < a.n_group; g0 += a.threads / width) {
      const int g = g0 + threadIdx.x / width;
      V v = {};
      if (g < a.n_group && at < many) v = load(g, at, all[(size_t)at * a.n_group + g]);
      for (int d = width / 2; d > 0; d >>= 1) v.add(v.across(d));
      if (at == 0 && g < a.n_group) end(g, v);
    }
    return;
  }
  __shared__ V parts[kGnThreads / 32][32];
  const int warp = threadIdx.x >> 5, warps = a.threads >> 5;
  int wide = 1;
  while (wide < a.n_group && wide < 32) wide *= 2;
  const int step = warps * (32 / wide);
  for (int g0 = 0; g0 < a.n_group; g0 += wide) {
    const int g = g0 + (lane & (wide - 1));
    V v = {};
    if (g < a.n_group)
      for (int i0 = warp * (32 / wide) + lane / wide; i0 < many; i0 += kGnPieces * step) {
        float2 p[kGnPieces];
#pragma unroll
        for (int k = 0; k < kGnPieces; ++k) p[k] = all[(size_t)min(i0 + k * step, many - 1) * a.n_group + g];
#pragma unroll
        for (int k = 0; k < kGnPieces; ++k)
          if (i0 + k * step < many) v.add(load(g, i0 + k * step, p[k]));
      }
    for (int d = wide; d < 32; d *= 2) v.add(v.across(d));
    if (lane < wide) parts[warp][lane] = v;
    __syncthreads();
    if ((int)threadIdx.x < wide && g < a.n_group) {
      for (int w = 1; w < warps; ++w) v.add(parts[w][lane]);
      end(g, v);
    }
    if (g0 + wide < a.n_group) __syncthreads();
  }
}

// mu and r of the walk's sample, from the partial results of its pieces, to shared memory; the block with its first row keeps them.
__device__ __forceinline__ void sample_stats(const GnArgs &a, const GnWalk &k, float *gs) {
  int first, many;
  sample_pieces(a, k, first, many);
  const float rows = (float)(k.hi - k.lo);
  sample_sums<GnMoments>(
      a, a.partial + (size_t)(first + k.s) * a.n_group * 2, many,
      [&](int g, int i, float2 p) { return GnMoments{(float)piece_rows(a, k, first + i), p.x, __fdividef(p.y, (float)a.t.group_copies[g])}; },
      [&](int g, const GnMoments &m) {
        const float2 r = {m.mean, 1.0f / sqrtf(m.sq / rows + a.eps)};
        *(float2 *)(gs + 2 * g) = r;
        if (first == (int)blockIdx.x) *(float2 *)(a.stats + ((size_t)k.s * a.n_group + g) * 2) = r;
      });
  __syncthreads();
}

// Second pass, forward.  The gates of a tile's rows are computed first, by all threads, into one of two buffers in turn: one wait a
// tile.
template <class T, class TO, int VEC, bool WHOLE, bool GATED>
__global__ void __launch_bounds__(kGnThreads, 1) gn_apply_kernel(GnArgs a) {
  after_previous();
  extern __shared__ __align__(128) char smem[];
  __shared__ alignas(8) uint64_t bars[2 * kGnStages];
  __shared__ volatile int abort_flag;
  GnRing ring;
  ring.open(a, blockIdx.x, smem, bars, &abort_flag, sizeof(T), 0);
  const int t = threadIdx.x;
  constexpr bool EXACT = sizeof(TO) == 4;
  float *gs = (float *)(smem + a.stages * a.stage_bytes);       // [n_group][2]
  float *gates = gs + 2 * a.n_group;                            // 2 x [tile][n_gate]
  const int slots = (a.c_out + VEC - 1) / VEC, R = a.threads / slots, ty = t / slots, ch = (t - ty * slots) * VEC, many = min(VEC, a.c_out - ch);
  const bool works = ty < R;
  TO *out = (TO *)a.out + ch;
  float w[VEC], b[VEC];
  int group[VEC], gate[VEC];
  bool mixed = false;                                           // scalars to be activated beside other channels
#pragma unroll
  for (int q = 0; q < VEC; ++q) {
    const int c = works && q < many ? ch + q : 0, sc = a.t.scalar_of_channel[c];
    group[q] = 2 * a.t.group_of_channel[c];
    w[q] = a.weight ? a.weight[a.t.field_of_channel[c]] : 1.f;
    b[q] = sc >= 0 && a.bias ? a.bias[sc] : 0.f;
    gate[q] = a.t.gate_of_channel[c];
    mixed |= (gate[q] == -1) != (gate[0] == -1);
  }
  // a thread's gate, every GR-th row
  const int GR = GATED ? a.threads / a.n_gate : 1, gj = GATED ? t % a.n_gate : 0, gr = GATED ? t / a.n_gate : 0;
  float gw = 1.f, gb = 0.f;
  int gg = 0;
  if (GATED) {
    const int c = a.c_out + gj, sc = a.t.scalar_of_channel[c];
    gg = 2 * a.t.group_of_channel[c];
    if (a.weight) gw = a.weight[a.t.field_of_channel[c]];
    if (a.bias) gb = a.bias[sc];
  }
  GnWalk walk;
  if (ring.r0 < ring.r1) walk.find(a, ring.r0);
  for (int row = ring.r0; row < ring.r1;) {
    const int end = min(walk.hi, ring.r1);
    const bool live = walk.live(a);
    float scale[VEC], shift[VEC], gscale = 0.f, gshift = 0.f;
    if (live) {
      sample_stats(a, walk, gs);
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        scale[q] = gs[group[q] + 1] * w[q];
        shift[q] = fmaf(-gs[group[q]], scale[q], b[q]);      // (mu itself is rounded by as much)
      }
      if (GATED) {
        gscale = gs[gg + 1] * gw;
        gshift = fmaf(-gs[gg], gscale, gb);
      }
    }
    while (row < end) {
      const T *tile = (const T *)ring.tile(a);
      const int first = ring.first, last = min(end, ring.end(a));
      if (GATED && live) {
        for (int i = row - first + gr; i < last - first; i += GR)
          if (gr < GR) {
            float z = fmaf((float)tile[i * a.c + a.c_out + gj], gscale, gshift);
            act_values<EXACT, 1>(&z, a.gate_act);
            gates[i * a.n_gate + gj] = z;
          }
        __syncthreads();
      }
      if (works) {
        for (int i = row - first + ty; i < last - first; i += 2 * R) {
          float v[2][VEC];
          const bool two = i + R < last - first;
          if (live) {
            load<T, VEC, WHOLE>(tile + i * a.c + ch, v[0], many);
            load<T, VEC, WHOLE>(tile + (two ? i + R : i) * a.c + ch, v[1], many);
            multiply_add<VEC>(v[0], v[0], (const float *)scale, (const float *)shift);
            multiply_add<VEC>(v[1], v[1], (const float *)scale, (const float *)shift);
            if (!mixed) {
              if (gate[0] == -1) act_values<EXACT, 2 * VEC>(&v[0][0], a.scalar_act);
            } else {
              float f[2 * VEC];
#pragma unroll
              for (int k = 0; k < 2 * VEC; ++k) f[k] = (&v[0][0])[k];
              act_values<EXACT, 2 * VEC>(f, a.scalar_act);
#pragma unroll
              for (int k = 0; k < 2 * VEC; ++k)
                if (gate[k % VEC] == -1) (&v[0][0])[k] = f[k];
            }
            if (GATED) {
#pragma unroll
              for (int q = 0; q < VEC; ++q)
                if (gate[q] >= 0) {
                  v[0][q] *= gates[i * a.n_gate + gate[q]];
                  v[1][q] *= gates[(two ? i + R : i) * a.n_gate + gate[q]];
                }
            }
          } else {
#pragma unroll
            for (int k = 0; k < 2 * VEC; ++k) (&v[0][0])[k] = 0.f;
          }
          store<TO, VEC, WHOLE>(out + (size_t)(first + i) * a.c_out, v[0], many);
          if (two) store<TO, VEC, WHOLE>(out + (size_t)(first + i + R) * a.c_out, v[1], many);
        }
      }
      ring.release(a, last);
      if (GATED) gates = gates == gs + 2 * a.n_group ? gates + a.tile * a.n_gate : gs + 2 * a.n_group;
      row = last;
    }
    if (live) __syncthreads();
    if (row < ring.r1) walk.place(a, row);
  }
  ring.close(a);
}

// Both backward passes.  SUMS: the sums of dz and dz xhat of each channel, as the groups' sums of a and a xhat of each piece and as the block's
// share of the parameters' gradients.  Else dx; the first blocks add up the parameters' gradients, kGnSum of them each.
// The gates of a tile's rows come first, by all threads: value, and (from the products with their fields) dz of the gate channels.
template <class T, int VEC, bool WHOLE, bool GATED, bool SUMS>
__global__ void __launch_bounds__(kGnThreads, 1) gn_bwd_kernel(GnArgs a, int sum_blocks) {
  after_previous();
  extern __shared__ __align__(128) char smem[];
  __shared__ alignas(8) uint64_t bars[2 * kGnStages];
  __shared__ volatile int abort_flag;
  const int t = threadIdx.x;
  if (!SUMS && (int)blockIdx.x < sum_blocks) {
    float *sm = (float *)smem;
    const int cols = a.n_field + a.n_scalar, col = blockIdx.x * kGnSum + (t & 31), part = t >> 5, parts = blockDim.x >> 5;
    float v = 0.f;
    if (col < cols)
      for (int i = part; i < a.blocks; i += parts) v += a.fields[(size_t)i * cols + col];
    sm[t] = v;
    __syncthreads();
    if (t < 32 && col < cols) {
      for (int p = 1; p < parts; ++p) v += sm[p * 32 + t];
      if (col < a.n_field) a.d_weight[col] = v;
      else a.d_bias[col - a.n_field] = v;
    }
    return;
  }
  const int block = SUMS ? (int)blockIdx.x : (int)blockIdx.x - sum_blocks;
  GnRing ring;
  ring.open(a, block, smem, bars, &abort_flag, sizeof(T), sizeof(T));
  constexpr bool EXACT = sizeof(T) == 4;
  const int slots = (a.c_out + VEC - 1) / VEC, R = a.threads / slots, ty = t / slots, ch = (t - ty * slots) * VEC, many = min(VEC, a.c_out - ch);
  const bool works = ty < R;
  const int GR = GATED ? min(a.threads / a.n_gate, max(R, kGnGateRows)) : 1, gj = GATED ? t % a.n_gate : 0, gr = GATED ? t / a.n_gate : 0;
  float *gs = (float *)(smem + a.stages * a.stage_bytes);       // !SUMS: [n_group][2]
  float *gates = gs + (SUMS ? 0 : 2 * a.n_group), *const gates0 = gates;      // 2 x [tile][n_gate]
  float *sums = gates0 + 2 * a.tile * a.n_gate;                 // SUMS: [max(R, GR)][c] twice, totals [c] twice
  const int RS = max(R, GR);
  float *tot = sums + 2 * RS * a.c;
  T *out = (T *)a.out + ch;
  float w[VEC], b[VEC];
  int group[VEC], gate[VEC];
  bool scalars = false;
  unsigned centred = 0;
#pragma unroll
  for (int q = 0; q < VEC; ++q) {
    const int c = works && q < many ? ch + q : 0, sc = a.t.scalar_of_channel[c];
    group[q] = a.t.group_of_channel[c];
    w[q] = a.weight ? a.weight[a.t.field_of_channel[c]] : 1.f;
    b[q] = sc >= 0 && a.bias ? a.bias[sc] : 0.f;
    gate[q] = a.t.gate_of_channel[c];
    scalars |= gate[q] == -1;
    centred |= (sc >= 0 ? 1u : 0u) << q;
  }
  float gw = 1.f, gb = 0.f, fw = 1.f;
  int gg = 0, gf = 0, flen = 0, fg = 0;                         // the gate's group; its field's first channel, length and group
  if (GATED) {
    const int c = a.c_out + gj, f = a.t.gate_field[gj];
    gg = a.t.group_of_channel[c];
    if (a.weight) gw = a.weight[a.t.field_of_channel[c]];
    if (a.bias) gb = a.bias[a.t.scalar_of_channel[c]];
    gf = a.t.field_first[f];
    flen = a.t.field_len[f];
    fg = a.t.group_of_channel[gf];
    if (a.weight) fw = a.weight[f];
  }
  if (SUMS)
    for (int i = t; i < 2 * a.c; i += a.threads) tot[i] = 0.f;
  GnWalk walk;
  if (ring.r0 < ring.r1) walk.find(a, ring.r0);
  for (int row = ring.r0; row < ring.r1;) {
    const int end = min(walk.hi, ring.r1);
    const bool live = walk.live(a);
    float mu[VEC], r[VEC], s1[VEC] = {}, s2[VEC] = {}, gmu = 0.f, gr_ = 0.f, fr = 0.f, g1 = 0.f, g2 = 0.f;
    if (live) {
      const float *st = a.stats + (size_t)walk.s * a.n_group * 2;
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        const float2 v = *(const float2 *)(st + 2 * group[q]);
        mu[q] = v.x;
        r[q] = v.y;
      }
      if (GATED) {
        gmu = st[2 * gg];
        gr_ = st[2 * gg + 1];
        fr = st[2 * fg + 1] * fw;
      }
      if (!SUMS) {
        int first, many;
        sample_pieces(a, walk, first, many);
        const float rows = (float)(walk.hi - walk.lo);
        sample_sums<GnSums>(
            a, a.partial + (size_t)(first + walk.s) * a.n_group * 2, many, [&](int, int, float2 p) { return GnSums{p.x, p.y}; },
            [&](int g, const GnSums &sum) {
              const float m = 1.0f / (rows * (float)a.t.group_copies[g]);
              gs[2 * g] = sum.u * m;
              gs[2 * g + 1] = sum.v * m;
            });
        __syncthreads();
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          s1[q] = centred >> q & 1 ? -gs[2 * group[q]] : 0.f;
          s2[q] = -gs[2 * group[q] + 1];
        }
        if (GATED) {
          g1 = gs[2 * gg];
          g2 = gs[2 * gg + 1];
        }
      }
    }
    while (row < end) {
      const char *stage = ring.tile(a);
      const T *tile = (const T *)stage, *grad = (const T *)(stage + a.x_bytes);
      const int first = ring.first, last = min(end, ring.end(a));
      if (GATED && live) {
        if (gr < GR)
          for (int i = row - first + gr; i < last - first; i += GR) {
            const float hat = ((float)tile[i * a.c + a.c_out + gj] - gmu) * gr_;
            float z = fmaf(hat, gw, gb), slope, p = 0.f;
            act_slopes<EXACT, 1>(&z, &slope, a.gate_act);
            gates[i * a.n_gate + gj] = z;
            for (int k = 0; k < flen; ++k) p = fmaf((float)tile[i * a.c + gf + k], (float)grad[i * a.c_out + gf + k], p);
            const float dz = p * fr * slope;
            if (SUMS) {
              g1 += dz;
              g2 = fmaf(dz, hat, g2);
            } else {
              ((T *)a.out)[(size_t)(first + i) * a.c + a.c_out + gj] = (T)(gr_ * (fmaf(dz, gw, -g1) - hat * g2));
            }
          }
        __syncthreads();
      }
      if (works && live) {
        for (int i = row - first + ty; i < last - first; i += 2 * R) {
          float hat[2][VEC], dz[2][VEC];
          const bool two = i + R < last - first;
          const int at[2] = {i, two ? i + R : i};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            load<T, VEC, WHOLE>(tile + at[u] * a.c + ch, hat[u], many);
            load<T, VEC, WHOLE>(grad + at[u] * a.c_out + ch, dz[u], many);
            multiply_add<VEC>(hat[u], mu, -1.f, hat[u]);
            multiply<VEC>(hat[u], hat[u], r);
          }
          if (scalars) {
            float z[2][VEC], slope[2][VEC];
#pragma unroll
            for (int u = 0; u < 2; ++u) multiply_add<VEC>(z[u], hat[u], w, b);
            act_slopes<EXACT, 2 * VEC>(&z[0][0], &slope[0][0], a.scalar_act);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int q = 0; q < VEC; ++q)
                if (gate[q] == -1) dz[u][q] *= slope[u][q];
          }
          if (GATED) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int q = 0; q < VEC; ++q)
                if (gate[q] >= 0) dz[u][q] *= gates[at[u] * a.n_gate + gate[q]];
          }
          if (SUMS) {
            multiply_add<VEC>(s1, s1, 1.f, dz[0]);
            multiply_add<VEC>(s2, dz[0], hat[0], s2);
            if (two) {
              multiply_add<VEC>(s1, s1, 1.f, dz[1]);
              multiply_add<VEC>(s2, dz[1], hat[1], s2);
            }
          } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // (s1 and s2 are negative here)
              multiply_add<VEC>(dz[u], dz[u], w, s1);
              multiply_add<VEC>(dz[u], hat[u], s2, dz[u]);
              multiply<VEC>(dz[u], dz[u], r);
              if (u == 0 || two) store<T, VEC, WHOLE>(out + (size_t)(first + at[u]) * a.c, dz[u], many);
            }
          }
        }
      }
      if (!SUMS && !live)
        for (long long i = (long long)row * a.c + t; i < (long long)last * a.c; i += a.threads) ((T *)a.out)[i] = (T)0.f;
      ring.release(a, last);
      if (GATED) gates = gates == gates0 ? gates + a.tile * a.n_gate : gates0;
      row = last;
    }
    if (SUMS && live) {
      float *second = sums + RS * a.c;
      for (int i = t; i < 2 * RS * a.c; i += a.threads) sums[i] = 0.f;
      __syncthreads();
      if (works) {
#pragma unroll
        for (int q = 0; q < VEC; ++q)
          if (q < many) {
            sums[ty * a.c + ch + q] = s1[q];
            second[ty * a.c + ch + q] = s2[q];
          }
      }
      if (GATED && gr < GR) {
        sums[gr * a.c + a.c_out + gj] = g1;
        second[gr * a.c + a.c_out + gj] = g2;
      }
      __syncthreads();
      for (int i = t; i < a.c; i += a.threads) {
        float u = 0.f, v = 0.f;
        for (int k = 0; k < RS; ++k) u += sums[k * a.c + i], v += second[k * a.c + i];
        sums[i] = u;
        second[i] = v;
        tot[i] += u;
        tot[a.c + i] += v;
      }
      __syncthreads();
      const int lane = t & 31;
      for (int g = t >> 5; g < a.n_group; g += a.threads >> 5) {
        const int from = a.t.group_first[g], len = a.t.group_len[g];
        float u = 0.f, v = 0.f;
        for (int i = lane; i < len; i += 32) {
          const float weight = a.weight ? a.weight[a.t.field_of_channel[from + i]] : 1.f;
          u = fmaf(weight, sums[from + i], u);
          v = fmaf(weight, second[from + i], v);
        }
        for (int d = 1; d < 32; d <<= 1) u += __shfl_xor_sync(0xffffffffu, u, d), v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == 0) *(float2 *)(a.partial + ((size_t)(block + walk.s) * a.n_group + g) * 2) = {u, v};
      }
    }
    if (live) __syncthreads();
    if (row < ring.r1) walk.place(a, row);
  }
  if (SUMS) {
    __syncthreads();
    float *p = a.fields + (size_t)block * (a.n_field + a.n_scalar);
    for (int f = t; f < a.n_field; f += a.threads) {
      const int from = a.t.field_first[f], len = a.t.field_len[f], sc = a.t.field_scalar[f];
      float v = 0.f;
      for (int i = 0; i < len; ++i) v += tot[a.c + from + i];
      p[f] = v;
      if (sc >= 0) p[a.n_field + sc] = tot[from];
    }
  }
  ring.close(a);
}

int type_bytes(int type) { return type == SSC_PREC_FP32 ? 4 : 2; }

// Channels to a thread: 16 bytes of them, four with their gradients (eight channels of two rows with gradients exceed a thread's 128 registers by 160 to 270
// bytes) and where rows are no multiple.  Gradients of bf16 rows by eight instead of four, both passes: 393216 rows of 128 with silu 105 and 115 us instead of 92 and 102,
// without an activation 65 and 93 instead of 71 and 82, 200000 of 128 + 24 with gates 157 and 135 instead of 86 and 93.
struct GnVec {
  int vec;
  bool whole;
};
GnVec gn_vec(int c, int c_out, int type, bool grads) {
  const int most = grads ? 4 : 16 / type_bytes(type);
  if (c % most == 0 && c_out % most == 0) return {most, true};
  return {4, c % 4 == 0 && c_out % 4 == 0};
}
constexpr int kGnBlocks = 2;               // to an SM

// Tiles of four rows to a thread, two where gradients come with them but no gates (8 to 16 KB, a multiple of 16 bytes); a ring of up to 88 KB.  (96011 rows of
// 64 + 12 channels: gradients with tiles of two rows 32 and 34 us, of four 29 and 30.  65536 of 256 without gates: two 40 and 40, four 43 and 41.)
void gn_shape(GnArgs &a, int type, int vec, bool grads) {
  const int bytes = a.c * type_bytes(type);
  const int wide = (a.c + vec - 1) / vec;
  a.threads = wide > 256 || a.n_gate > 256 ? kGnThreads : 256;
  const int rows = a.threads / wide;
  const long long slots = (long long)sm_count() * kGnBlocks;
  int each = grads && a.n_gate == 0 ? 2 : 4;
  while (each > 1 && a.n <= slots * rows * (each / 2)) each /= 2;       // (few rows: more blocks; 3501 of 32 + 6 channels 9.9 us, 12.7 without)
  while ((rows * each * bytes) % 16 || (rows * each * a.c_out * type_bytes(type)) % 16) each *= 2;
  a.tile = rows * each;
  a.x_bytes = (uint32_t)align_up((size_t)a.tile * bytes, 128);
  a.stage_bytes = a.x_bytes + (grads ? (uint32_t)align_up((size_t)a.tile * a.c_out * type_bytes(type), 128) : 0);
  a.stages = (int)(90112 / a.stage_bytes);
  if (a.stages > kGnStages) a.stages = kGnStages;
  if (a.stages < 2) a.stages = 2;
  const long long tiles = ((long long)a.n + a.tile - 1) / a.tile, per = (tiles + slots - 1) / slots;
  a.range = (int)(per * a.tile);
  a.blocks = (int)((tiles + per - 1) / per);
}

size_t gn_scratch(int batch, int n_group, int n_cols) {
  const size_t blocks = (size_t)sm_count() * kGnBlocks;
  return ((blocks + batch) * 2 * (size_t)n_group + blocks * (size_t)n_cols) * sizeof(float) + 16;
}

int gn_fill(GnArgs &a, const int32_t *table, const char *what) {
  SSC_REQUIRE(a.n >= 0 && a.n <= 1 << 30 && a.batch >= 1 && a.c >= 1 && a.c_out >= 1 && a.n_gate >= 0 && a.c_out + a.n_gate == a.c, "%s: bad sizes", what);
  SSC_REQUIRE(a.n_group >= 1 && a.n_group <= a.c && a.n_field >= 1 && a.n_field <= a.c && a.n_scalar >= 0 && a.n_scalar <= a.n_field, "%s: bad layout", what);
  SSC_REQUIRE(a.scalar_act >= 0 && a.scalar_act <= 4 && a.gate_act >= 0 && a.gate_act <= 4, "%s: unknown activation", what);
  SSC_REQUIRE(a.eps > 0.f, "%s: eps must be positive", what);
  SSC_REQUIRE(table && a.offsets && a.stats && (a.n == 0 || (a.x && a.out)), "%s: null pointer", what);
  SSC_REQUIRE((((uintptr_t)a.x | (uintptr_t)a.gy | (uintptr_t)a.out) & 15) == 0, "%s: rows must start at a multiple of 16 bytes", what);
  const int32_t *p = table;
  a.t.group_of_channel = p; p += a.c;
  a.t.field_of_channel = p; p += a.c;
  a.t.scalar_of_channel = p; p += a.c;
  a.t.gate_of_channel = p; p += a.c_out;
  a.t.field_first = p; p += a.n_field;
  a.t.field_len = p; p += a.n_field;
  a.t.field_scalar = p; p += a.n_field;
  a.t.gate_field = p; p += a.n_gate;
  a.t.group_first = p; p += a.n_group;
  a.t.group_len = p; p += a.n_group;
  a.t.group_copies = p;
  a.alarm = alarm_word();
  return SSC_OK;
}

template <class T, class TO, int VEC, bool WHOLE>
cudaError_t gn_fwd(const GnArgs &a, cudaStream_t st) {
  const dim3 block(a.threads), grid(a.blocks);
  const size_t ring = (size_t)a.stages * a.stage_bytes, rows = a.threads / ((a.c + VEC - 1) / VEC);
  const size_t stats = ring + 2 * (rows + 1) * a.c * sizeof(float), room = ring + (2 * (size_t)a.n_group + 2 * (size_t)a.tile * a.n_gate) * sizeof(float);
  auto apply = a.n_gate ? gn_apply_kernel<T, TO, VEC, WHOLE, true> : gn_apply_kernel<T, TO, VEC, WHOLE, false>;
  cudaError_t e = allow_smem((const void *)gn_stats_kernel<T, VEC, WHOLE>, stats);
  if (e == cudaSuccess) e = allow_smem((const void *)apply, room);
  if (e == cudaSuccess) e = launch_ready(gn_stats_kernel<T, VEC, WHOLE>, grid, block, stats, st, a);
  return e == cudaSuccess ? launch_ready(apply, grid, block, room, st, a) : e;
}

template <class T, int VEC, bool WHOLE>
cudaError_t gn_bwd(const GnArgs &a, cudaStream_t st) {
  const dim3 block(a.threads);
  const size_t ring = (size_t)a.stages * a.stage_bytes;
  size_t rows = a.threads / ((a.c_out + VEC - 1) / VEC);
  if (a.n_gate && rows < (size_t)kGnGateRows) rows = kGnGateRows;
  const size_t gates = 2 * (size_t)a.tile * a.n_gate;
  const size_t first = ring + (gates + 2 * (rows + 1) * a.c) * sizeof(float), second = ring + (gates + 2 * (size_t)a.n_group) * sizeof(float);
  auto one = a.n_gate ? gn_bwd_kernel<T, VEC, WHOLE, true, true> : gn_bwd_kernel<T, VEC, WHOLE, false, true>;
  auto two = a.n_gate ? gn_bwd_kernel<T, VEC, WHOLE, true, false> : gn_bwd_kernel<T, VEC, WHOLE, false, false>;
  cudaError_t e = allow_smem((const void *)one, first);
  if (e == cudaSuccess) e = allow_smem((const void *)two, second);
  const int sum_blocks = ceil_div(a.n_field + a.n_scalar, kGnSum);
  if (e == cudaSuccess) e = launch_ready(one, dim3(a.blocks), block, first, st, a, 0);
  return e == cudaSuccess ? launch_ready(two, dim3(a.blocks + sum_blocks), block, second, st, a, sum_blocks) : e;
}

template <class T, class TO>
cudaError_t gn_fwd_vec(const GnArgs &a, GnVec v, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (v.vec == 8) return gn_fwd<T, TO, 8, true>(a, st);
  return v.whole ? gn_fwd<T, TO, 4, true>(a, st) : gn_fwd<T, TO, 4, false>(a, st);
}
template <class T>
cudaError_t gn_bwd_vec(const GnArgs &a, GnVec v, cudaStream_t st) {
  return v.whole ? gn_bwd<T, 4, true>(a, st) : gn_bwd<T, 4, false>(a, st);
}
bool known_type(int t) { return t == SSC_PREC_FP32 || t == SSC_PREC_F16 || t == SSC_PREC_BF16; }

}  // namespace
}  // namespace ssc

extern "C" size_t ssc_group_norm_scratch_bytes(int batch, int n_group, int n_field, int n_scalar) {
  if (batch < 1 || n_group < 0 || n_field < 0 || n_scalar < 0) return 0;
  return ssc::gn_scratch(batch, n_group, n_field + n_scalar);
}

extern "C" int ssc_group_norm_fwd(const void *x, int type, int n, int c, const int32_t *offsets, int batch, const int32_t *table, int n_field,
                                  int n_scalar, int n_group, int n_gate, const float *weight, const float *bias, float eps, int scalar_act, int gate_act,
                                  void *out, int out_type, float *stats, int32_t *status, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace ssc;
  SSC_REQUIRE(known_type(type) && known_type(out_type) && (type == out_type || type == SSC_PREC_FP32), "group_norm_fwd: unknown types");
  GnArgs a = {};
  a.x = x; a.out = out; a.n = n; a.c = c; a.c_out = c - n_gate; a.n_gate = n_gate; a.n_group = n_group; a.n_field = n_field; a.n_scalar = n_scalar;
  a.batch = batch; a.offsets = offsets; a.weight = weight; a.bias = bias; a.eps = eps; a.scalar_act = scalar_act; a.gate_act = gate_act; a.stats = stats;
  a.status = status;
  if (int e = gn_fill(a, table, "group_norm_fwd")) return e;
  if (n == 0) return SSC_OK;
  const GnVec vec = gn_vec(c, a.c_out, type, false);
  SSC_REQUIRE(n_gate <= kGnThreads, "group_norm_fwd: %d gates, at most %d", n_gate, kGnThreads);
  SSC_REQUIRE(c <= 4 * kGnThreads, "group_norm_fwd: %d channels, at most %d", c, 4 * kGnThreads);
  gn_shape(a, type, vec.vec, false);
  if (scratch == nullptr || ((uintptr_t)scratch & 15) != 0 || scratch_bytes < gn_scratch(batch, n_group, 0)) return fail(SSC_ERR_SCRATCH, "group_norm_fwd: scratch too small");
  a.partial = (float *)scratch;
  const cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (type == SSC_PREC_F16) e = gn_fwd_vec<__half, __half>(a, vec, st);
  else if (type == SSC_PREC_BF16) e = gn_fwd_vec<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
  else if (out_type == SSC_PREC_F16) e = gn_fwd_vec<float, __half>(a, vec, st);
  else if (out_type == SSC_PREC_BF16) e = gn_fwd_vec<float, __nv_bfloat16>(a, vec, st);
  else e = gn_fwd_vec<float, float>(a, vec, st);
  if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "group_norm_fwd: %s", cudaGetErrorString(e));
  note_launches(2);
  SSC_CHECK_LAUNCH("group_norm_fwd");
  return SSC_OK;
}

extern "C" int ssc_group_norm_bwd(const void *x, const void *gy, int type, int n, int c, const int32_t *offsets, int batch, const int32_t *table,
                                  int n_field, int n_scalar, int n_group, int n_gate, const float *weight, const float *bias, float eps, int scalar_act,
                                  int gate_act, const float *stats, void *gx, float *d_weight, float *d_bias, int32_t *status, void *scratch,
                                  size_t scratch_bytes, void *stream) {
  using namespace ssc;
  SSC_REQUIRE(known_type(type), "group_norm_bwd: unknown type");
  GnArgs a = {};
  a.x = x; a.gy = gy; a.out = gx; a.n = n; a.c = c; a.c_out = c - n_gate; a.n_gate = n_gate; a.n_group = n_group; a.n_field = n_field;
  a.n_scalar = n_scalar; a.batch = batch; a.offsets = offsets; a.weight = weight; a.bias = bias; a.eps = eps; a.scalar_act = scalar_act;
  a.gate_act = gate_act; a.stats = const_cast<float *>(stats); a.d_weight = d_weight; a.d_bias = d_bias; a.status = status;
  if (int e = gn_fill(a, table, "group_norm_bwd")) return e;
  SSC_REQUIRE((n == 0 || gy) && d_weight && (n_scalar == 0 || d_bias), "group_norm_bwd: null pointer");
  const cudaStream_t st = as_stream(stream);
  if (n == 0) {
    cudaError_t e = cudaMemsetAsync(d_weight, 0, n_field * sizeof(float), st);
    if (e == cudaSuccess && n_scalar) e = cudaMemsetAsync(d_bias, 0, n_scalar * sizeof(float), st);
    if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "group_norm_bwd: %s", cudaGetErrorString(e));
    return SSC_OK;
  }
  const GnVec vec = gn_vec(c, a.c_out, type, true);
  SSC_REQUIRE(n_gate <= kGnThreads, "group_norm_bwd: %d gates, at most %d", n_gate, kGnThreads);
  SSC_REQUIRE(c <= 4 * kGnThreads, "group_norm_bwd: %d channels, at most %d", c, 4 * kGnThreads);
  gn_shape(a, type, vec.vec, true);
  if (scratch == nullptr || ((uintptr_t)scratch & 15) != 0 || scratch_bytes < gn_scratch(batch, n_group, n_field + n_scalar))
    return fail(SSC_ERR_SCRATCH, "group_norm_bwd: scratch too small");
  a.partial = (float *)scratch;
  a.fields = a.partial + 2 * ((size_t)a.blocks + batch) * n_group;
  cudaError_t e = type == SSC_PREC_F16 ? gn_bwd_vec<__half>(a, vec, st) : type == SSC_PREC_BF16 ? gn_bwd_vec<__nv_bfloat16>(a, vec, st) : gn_bwd_vec<float>(a, vec, st);
  if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "group_norm_bwd: %s", cudaGetErrorString(e));
  note_launches(2);
  SSC_CHECK_LAUNCH("group_norm_bwd");
  return SSC_OK;
}
