// Group norm of the rows of ragged samples (channels last) with the gated activation behind it, and its gradients.
//
// A group is a range of channels, the copies of fields of one order; its statistics run over the rows of a sample and the
// copies.  Scalars: mu = mean, v = mean (x - mu)^2.  Fields of order l > 0: mu = 0, v = mean |x|^2, which commutes with
// rotations.  With r = (v + eps)^-1/2: z = (x - mu) r w + b; the activation follows.  Backward, with a = dz w, xhat = (x - mu) r and M =
// rows * copies: dx = r (a - [scalars] sum(a) / M - xhat sum(a xhat) / M), dw = sum dz xhat, db = sum dz.
//
// Memory-bound: each direction is two passes over the rows, sums first.  The samples are cut into chunks of equal length,
// one to a block, about four blocks to an SM; a block leaves one partial result for each group, and every block of the second pass adds up
// those of its own sample in a fixed order (no atomics: the same bits every time).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ssc_common.cuh"
#include "ssc_rows_act.cuh"

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
  int chunk_rows, max_chunks;
  float *partial;      // [max_chunks][n_group][2]
  float *fields;       // [max_chunks][n_field + n_scalar]
  float *stats;        // [batch][n_group][2]: mu, r
  float *d_weight, *d_bias;
};

constexpr int kGnThreads = 512;             // at most; 256 where a row has fewer slots than that
constexpr int kGnSum = 32;                  // columns of d_weight | d_bias to a block of the second backward pass

struct Chunk {
  int sample;        // -1: rows of no sample, -2: nothing
  int lo, hi;        // rows
  int first, chunks; // the sample's chunks
  int rows;          // of the sample
  int total;         // chunks of all samples
};

// The chunk of block b: samples are cut one after the other, the rows before the first and behind the last one come last.
// Offsets beyond the rows are cut down to them.  Called by the whole block.
__device__ __forceinline__ Chunk find_chunk(const GnArgs &a, int b, Chunk *shared) {
  if (threadIdx.y == 0 && threadIdx.x == 0) shared->sample = -2;
  const int t = threadIdx.y * blockDim.x + threadIdx.x;
  __syncthreads();
  if (t < 32) {
    int base = 0, edge0 = 0, edge1 = 0;
    for (int s0 = 0; s0 < a.batch; s0 += 32) {
      const int s = s0 + t;
      int lo = 0, hi = 0;
      if (s < a.batch) {
        lo = min(max(a.offsets[s], 0), a.n);
        hi = min(max(a.offsets[s + 1], lo), a.n);
        if (s == 0) edge0 = lo;
        if (s == a.batch - 1) edge1 = hi;
      }
      const int mine = (int)(((long long)(hi - lo) + a.chunk_rows - 1) / a.chunk_rows);
      int upto = mine;
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, d);
        if (t >= d) upto += v;
      }
      const int first = base + upto - mine;
      if (b >= first && b < first + mine) {
        shared->sample = s;
        shared->lo = lo + (b - first) * a.chunk_rows;
        shared->hi = min(shared->lo + a.chunk_rows, hi);
        shared->first = first;
        shared->chunks = mine;
        shared->rows = hi - lo;
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
    edge0 = __shfl_sync(0xffffffffu, edge0, 0);
    edge1 = __shfl_sync(0xffffffffu, edge1, (a.batch - 1) & 31);
    if (t == 0) {
      shared->total = min(base, a.max_chunks);
      if (b >= base) {
        const int before = (int)(((long long)edge0 + a.chunk_rows - 1) / a.chunk_rows), k = b - base;
        const int lo = k < before ? k * a.chunk_rows : edge1 + (k - before) * a.chunk_rows;
        const int end = k < before ? edge0 : a.n;
        if (lo >= 0 && lo < end) {
          shared->sample = -1;
          shared->lo = lo;
          shared->hi = min(lo + a.chunk_rows, end);
        }
      }
    }
  }
  __syncthreads();
  return *shared;
}

// Rows of T, VEC channels at a time.
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };
template <class T, int VEC>
__device__ __forceinline__ void load(const T *p, float *v) {
  const Pack<T, VEC> k = *(const Pack<T, VEC> *)p;
#pragma unroll
  for (int q = 0; q < VEC; ++q) v[q] = (float)k.v[q];
}
template <class T, int VEC>
__device__ __forceinline__ void store(T *p, const float *v) {
  Pack<T, VEC> k;
#pragma unroll
  for (int q = 0; q < VEC; ++q) k.v[q] = (T)v[q];
  *(Pack<T, VEC> *)p = k;
}

// Two sets of values as (count, mean, sum of squared distances from it), added to one (Chan et al. 1979).  Sums of squares and
// of values alone would lose the variance of rows far from zero.
__device__ __forceinline__ void merge(float &n, float &m, float &q, float n2, float m2, float q2) {
  const float tot = n + n2;
  if (tot <= 0.f) return;
  const float f = __fdividef(n2, tot), d = m2 - m;
  m = fmaf(d, f, m);
  q += q2 + d * d * n * f;
  n = tot;
}

// First pass, forward: mean and sum of squared distances of each group of a chunk.  A thread takes four rows at a time, exactly
// (mean first), and adds them to its running values.
template <class T, int VEC>
__global__ void __launch_bounds__(kGnThreads) gn_stats_kernel(GnArgs a) {
  after_previous();
  __shared__ Chunk shared;
  extern __shared__ float sm[];                       // [R][c] means, [R][c] squares
  const Chunk k = find_chunk(a, blockIdx.x, &shared);
  if (k.sample < 0) return;
  const int R = blockDim.y, ty = threadIdx.y, ch = threadIdx.x * VEC;
  float mean[VEC], sq[VEC], centred[VEC];
#pragma unroll
  for (int q = 0; q < VEC; ++q) {
    mean[q] = sq[q] = 0.f;
    centred[q] = a.t.scalar_of_channel[ch + q] >= 0 ? 1.f : 0.f;
  }
  const T *x = (const T *)a.x + ch;
  int row = k.lo + ty;
  float have = 0.f;
  for (; row + 3 * R < k.hi; row += 4 * R) {
    float v[4][VEC];
#pragma unroll
    for (int u = 0; u < 4; ++u) load<T, VEC>(x + (size_t)(row + u * R) * a.c, v[u]);
    const float f = __fdividef(4.f, have + 4.f);
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      const float mb = ((v[0][q] + v[1][q]) + (v[2][q] + v[3][q])) * (0.25f * centred[q]);
      float s = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) s = fmaf(v[u][q] - mb, v[u][q] - mb, s);
      const float d = mb - mean[q];
      mean[q] = fmaf(d, f, mean[q]);
      sq[q] += fmaf(d * d, have * f, s);
    }
    have += 4.f;
  }
  for (; row < k.hi; row += R) {
    float v[VEC];
    load<T, VEC>(x + (size_t)row * a.c, v);
    const float f = __fdividef(1.f, have + 1.f);
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      const float mb = v[q] * centred[q], d = mb - mean[q], e = v[q] - mb;
      mean[q] = fmaf(d, f, mean[q]);
      sq[q] += fmaf(d * d, have * f, e * e);
    }
    have += 1.f;
  }
  float *sq_s = sm + R * a.c;
#pragma unroll
  for (int q = 0; q < VEC; ++q) {
    sm[ty * a.c + ch + q] = mean[q];
    sq_s[ty * a.c + ch + q] = sq[q];
  }
  __syncthreads();
  const int t = ty * blockDim.x + threadIdx.x, threads = blockDim.x * R, rows = k.hi - k.lo;
  for (int i = t; i < a.c; i += threads) {
    float n = 0.f, m = 0.f, s = 0.f;
    for (int r = 0; r < R; ++r)
      if (r < rows) merge(n, m, s, (float)((rows - r + R - 1) / R), sm[r * a.c + i], sq_s[r * a.c + i]);
    sm[i] = m;
    sq_s[i] = s;
  }
  __syncthreads();
  const int lane = t & 31, warps = threads >> 5;      // (the whole ones; a block has more than 128 threads)
  if (t < warps * 32)
    for (int g = t >> 5; g < a.n_group; g += warps) {
      const int first = a.t.group_first[g], len = a.t.group_len[g];
      float n = 0.f, m = 0.f, s = 0.f;
      for (int i = lane; i < len; i += 32) merge(n, m, s, (float)rows, sm[first + i], sq_s[first + i]);
      for (int d = 1; d < 32; d <<= 1) {
        const float n2 = __shfl_down_sync(0xffffffffu, n, d), m2 = __shfl_down_sync(0xffffffffu, m, d), s2 = __shfl_down_sync(0xffffffffu, s, d);
        merge(n, m, s, n2, m2, s2);
      }
      if (lane == 0) {
        float *p = a.partial + ((size_t)blockIdx.x * a.n_group + g) * 2;
        p[0] = m;
        p[1] = s;
      }
    }
}

// mu and r of the block's sample, from the partial results of its chunks, to shared memory; the first chunk's block keeps them.
__device__ __forceinline__ void sample_stats(const GnArgs &a, const Chunk &k, float *gs) {
  const int t = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  const int lane = t & 31, warps = threads >> 5;
  if (t < warps * 32)
    for (int g = t >> 5; g < a.n_group; g += warps) {
      const float copies = (float)a.t.group_copies[g];
      float n = 0.f, m = 0.f, s = 0.f;
      for (int i = lane; i < k.chunks && k.first + i < a.max_chunks; i += 32) {
        const float *p = a.partial + ((size_t)(k.first + i) * a.n_group + g) * 2;
        merge(n, m, s, (float)min(a.chunk_rows, k.rows - i * a.chunk_rows) * copies, p[0], p[1]);
      }
      for (int d = 1; d < 32; d <<= 1) {
        const float n2 = __shfl_down_sync(0xffffffffu, n, d), m2 = __shfl_down_sync(0xffffffffu, m, d), s2 = __shfl_down_sync(0xffffffffu, s, d);
        merge(n, m, s, n2, m2, s2);
      }
      if (lane == 0) {
        const float r = 1.0f / sqrtf(s / ((float)k.rows * copies) + a.eps);
        gs[2 * g] = m;
        gs[2 * g + 1] = r;
        if (k.first == (int)blockIdx.x) {
          a.stats[((size_t)k.sample * a.n_group + g) * 2] = m;
          a.stats[((size_t)k.sample * a.n_group + g) * 2 + 1] = r;
        }
      }
    }
  __syncthreads();
}

// Second pass, forward.  Gates go through shared memory, two buffers in turn: one wait for four rows of a thread.
template <class T, class TO, int VEC, bool GATED>
__global__ void __launch_bounds__(kGnThreads) gn_apply_kernel(GnArgs a) {
  after_previous();
  __shared__ Chunk shared;
  extern __shared__ float sm[];                       // [n_group][2], gates: 2 x [4 R][n_gate]
  const Chunk k = find_chunk(a, blockIdx.x, &shared);
  if (k.sample == -2) return;
  const int R = blockDim.y, ty = threadIdx.y, ch = threadIdx.x * VEC;
  const bool body = ch < a.c_out;
  TO *out = (TO *)a.out + ch;
  if (k.sample < 0) {                                 // rows of no sample
    const float zero[VEC] = {};
    if (body)
      for (int row = k.lo + ty; row < k.hi; row += R) store<TO, VEC>(out + (size_t)row * a.c_out, zero);
    return;
  }
  sample_stats(a, k, sm);
  float mu[VEC], scale[VEC], shift[VEC];
  int gate[VEC];
#pragma unroll
  for (int q = 0; q < VEC; ++q) {
    const int g = a.t.group_of_channel[ch + q], sc = a.t.scalar_of_channel[ch + q];
    mu[q] = sm[2 * g];
    scale[q] = sm[2 * g + 1] * (a.weight ? a.weight[a.t.field_of_channel[ch + q]] : 1.f);
    shift[q] = sc >= 0 && a.bias ? a.bias[sc] : 0.f;
    gate[q] = body ? a.t.gate_of_channel[ch + q] : -2;
  }
  bool mixed = false;                                 // scalars to be activated beside other channels
#pragma unroll
  for (int q = 1; q < VEC; ++q) mixed |= (gate[q] == -1) != (gate[0] == -1);
  constexpr bool EXACT = sizeof(TO) == 4;
  const T *x = (const T *)a.x + ch;
  float *gates = sm + 2 * a.n_group;
  for (int row0 = k.lo; row0 < k.hi; row0 += 4 * R) {
    float v[4][VEC];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = row0 + u * R + ty;
      if (row < k.hi) {
        load<T, VEC>(x + (size_t)row * a.c, v[u]);
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[u][q] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int q = 0; q < VEC; ++q) v[u][q] = fmaf(v[u][q] - mu[q], scale[q], shift[q]);
    if (GATED) {
      if (!body) {
        act_values<EXACT, 4 * VEC>(&v[0][0], a.gate_act);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int q = 0; q < VEC; ++q) gates[(u * R + ty) * a.n_gate + ch - a.c_out + q] = v[u][q];
      }
      __syncthreads();
    }
    if (body) {
      if (!mixed) {
        if (gate[0] == -1) act_values<EXACT, 4 * VEC>(&v[0][0], a.scalar_act);
      } else {
        float f[4 * VEC];
#pragma unroll
        for (int i = 0; i < 4 * VEC; ++i) f[i] = (&v[0][0])[i];
        act_values<EXACT, 4 * VEC>(f, a.scalar_act);
#pragma unroll
        for (int i = 0; i < 4 * VEC; ++i)
          if (gate[i % VEC] == -1) (&v[0][0])[i] = f[i];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = row0 + u * R + ty;
        if (row >= k.hi) continue;
        if (GATED) {
#pragma unroll
          for (int q = 0; q < VEC; ++q)
            if (gate[q] >= 0) v[u][q] *= gates[(u * R + ty) * a.n_gate + gate[q]];
        }
        store<TO, VEC>(out + (size_t)row * a.c_out, v[u]);
      }
    }
    if (GATED) gates = gates == sm + 2 * a.n_group ? gates + 4 * R * a.n_gate : sm + 2 * a.n_group;
  }
}

// dz and xhat of two rows of a thread; products with the gates' fields go through shared memory.
template <class T, int VEC, bool GATED>
struct GnBack {
  float mu[VEC], r[VEC], w[VEC], b[VEC];
  int gate[VEC];
  int first[VEC], len[VEC];      // gate channels: the field behind the gate
  bool scalars;                  // some channel has the scalar activation
  float *gates, *prods;          // [2 R][n_gate], [2 R][c_out]

  __device__ __forceinline__ void setup(const GnArgs &a, const Chunk &k, int ch, float *room) {
    const bool body = ch < a.c_out;
    scalars = false;
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      const int g = a.t.group_of_channel[ch + q], sc = a.t.scalar_of_channel[ch + q];
      const float *s = a.stats + ((size_t)k.sample * a.n_group + g) * 2;
      mu[q] = s[0];
      r[q] = s[1];
      w[q] = a.weight ? a.weight[a.t.field_of_channel[ch + q]] : 1.f;
      b[q] = sc >= 0 && a.bias ? a.bias[sc] : 0.f;
      gate[q] = body ? a.t.gate_of_channel[ch + q] : -2;
      scalars |= gate[q] == -1;
      if (GATED) {
        const int f = body ? 0 : a.t.gate_field[ch - a.c_out + q];
        first[q] = body ? 0 : a.t.field_first[f];
        len[q] = body ? 0 : a.t.field_len[f];
      }
    }
    gates = room;
    prods = room + 2 * blockDim.y * a.n_gate;
  }
  // (called by the whole block; rows behind the chunk's end give zeros)
  __device__ __forceinline__ void rows(const GnArgs &a, const Chunk &k, int row0, int ch, float (&hat)[2][VEC], float (&dz)[2][VEC]) {
    const int R = blockDim.y, ty = threadIdx.y;
    const bool body = ch < a.c_out;
    constexpr bool EXACT = sizeof(T) == 4;
    float z[2][VEC], slope[2][VEC];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = row0 + u * R + ty;
      const bool live = row < k.hi;
#pragma unroll
      for (int q = 0; q < VEC; ++q) hat[u][q] = mu[q], dz[u][q] = 0.f;
      if (live) load<T, VEC>((const T *)a.x + (size_t)row * a.c + ch, hat[u]);
      if (live && body) load<T, VEC>((const T *)a.gy + (size_t)row * a.c_out + ch, dz[u]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        hat[u][q] = (hat[u][q] - mu[q]) * r[q];
        z[u][q] = fmaf(hat[u][q], w[q], b[q]);
      }
    if (GATED && body) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < VEC; ++q) prods[(u * R + ty) * a.c_out + ch + q] = dz[u][q] * z[u][q];
    }
    if (!body || scalars) act_slopes<EXACT, 2 * VEC>(&z[0][0], &slope[0][0], body ? a.scalar_act : a.gate_act);
    if (GATED) {
      if (!body) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int q = 0; q < VEC; ++q) gates[(u * R + ty) * a.n_gate + ch - a.c_out + q] = z[u][q];
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int at = u * R + ty;
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        if (gate[q] == -1) dz[u][q] *= slope[u][q];
        else if (GATED && gate[q] >= 0) dz[u][q] *= gates[at * a.n_gate + gate[q]];
        else if (GATED && !body) {
          float s = 0.f;
          for (int i = 0; i < len[q]; ++i) s += prods[at * a.c_out + first[q] + i];
          dz[u][q] = row0 + at < k.hi ? s * slope[u][q] : 0.f;
        }
      }
    }
    if (GATED) __syncthreads();
  }
};

// First pass, backward: sum of dz and of dz xhat of each channel of a chunk, as the groups' sums of a and a xhat and as the
// chunk's share of the parameters' gradients.
template <class T, int VEC, bool GATED>
__global__ void __launch_bounds__(kGnThreads) gn_bwd_sums_kernel(GnArgs a) {
  after_previous();
  __shared__ Chunk shared;
  extern __shared__ float sm[];                       // [R][c], [R][c]; before that the gates and products of GnBack
  const Chunk k = find_chunk(a, blockIdx.x, &shared);
  if (k.sample < 0) return;
  const int R = blockDim.y, ty = threadIdx.y, ch = threadIdx.x * VEC;
  GnBack<T, VEC, GATED> back;
  back.setup(a, k, ch, sm);
  float s1[VEC] = {}, s2[VEC] = {};
  for (int row0 = k.lo; row0 < k.hi; row0 += 2 * R) {
    float hat[2][VEC], dz[2][VEC];
    back.rows(a, k, row0, ch, hat, dz);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        s1[q] += dz[u][q];
        s2[q] = fmaf(dz[u][q], hat[u][q], s2[q]);
      }
  }
  float *s2_s = sm + R * a.c;
#pragma unroll
  for (int q = 0; q < VEC; ++q) {
    sm[ty * a.c + ch + q] = s1[q];
    s2_s[ty * a.c + ch + q] = s2[q];
  }
  __syncthreads();
  const int t = ty * blockDim.x + threadIdx.x, threads = blockDim.x * R;
  for (int i = t; i < a.c; i += threads) {
    float u = 0.f, v = 0.f;
    for (int r = 0; r < R; ++r) u += sm[r * a.c + i], v += s2_s[r * a.c + i];
    sm[i] = u;
    s2_s[i] = v;
  }
  __syncthreads();
  for (int f = t; f < a.n_field; f += threads) {
    float *p = a.fields + (size_t)blockIdx.x * (a.n_field + a.n_scalar);
    const int first = a.t.field_first[f], len = a.t.field_len[f], sc = a.t.field_scalar[f];
    float v = 0.f;
    for (int i = 0; i < len; ++i) v += s2_s[first + i];
    p[f] = v;
    if (sc >= 0) p[a.n_field + sc] = sm[first];
  }
  const int lane = t & 31, warps = threads >> 5;
  if (t < warps * 32)
    for (int g = t >> 5; g < a.n_group; g += warps) {
      const int first = a.t.group_first[g], len = a.t.group_len[g];
      float u = 0.f, v = 0.f;
      for (int i = lane; i < len; i += 32) {
        const float w = a.weight ? a.weight[a.t.field_of_channel[first + i]] : 1.f;
        u = fmaf(w, sm[first + i], u);
        v = fmaf(w, s2_s[first + i], v);
      }
      for (int d = 1; d < 32; d <<= 1) u += __shfl_xor_sync(0xffffffffu, u, d), v += __shfl_xor_sync(0xffffffffu, v, d);
      if (lane == 0) {
        float *p = a.partial + ((size_t)blockIdx.x * a.n_group + g) * 2;
        p[0] = u;
        p[1] = v;
      }
    }
}

// Second pass, backward: dx.  The first blocks add up the parameters' gradients, kGnSum of them each.
template <class T, int VEC, bool GATED>
__global__ void __launch_bounds__(kGnThreads) gn_bwd_apply_kernel(GnArgs a, int sum_blocks) {
  after_previous();
  __shared__ Chunk shared;
  extern __shared__ float sm[];                       // [n_group][2], gates and products; or [threads] sums
  const int R = blockDim.y, ty = threadIdx.y, ch = threadIdx.x * VEC;
  const int t = ty * blockDim.x + threadIdx.x, threads = blockDim.x * R;
  const Chunk k = find_chunk(a, (int)blockIdx.x - sum_blocks, &shared);
  if ((int)blockIdx.x < sum_blocks) {
    const int cols = a.n_field + a.n_scalar, lanes = min(kGnSum, threads), parts = threads / lanes;
    for (int c0 = blockIdx.x * kGnSum; c0 < min((int)(blockIdx.x + 1) * kGnSum, cols); c0 += lanes) {
      const int col = c0 + t % lanes, part = t / lanes;
      float v = 0.f;
      if (part < parts && col < cols)
        for (int i = part; i < shared.total; i += parts) v += a.fields[(size_t)i * cols + col];
      __syncthreads();
      sm[t] = v;
      __syncthreads();
      if (t < lanes && col < cols) {
        for (int p = 1; p < parts; ++p) v += sm[p * lanes + t];
        if (col < a.n_field) a.d_weight[col] = v;
        else a.d_bias[col - a.n_field] = v;
      }
    }
    return;
  }
  if (k.sample == -2) return;
  T *out = (T *)a.out + ch;
  if (k.sample < 0) {
    const float zero[VEC] = {};
    for (int row = k.lo + ty; row < k.hi; row += R) store<T, VEC>(out + (size_t)row * a.c, zero);
    return;
  }
  const int lane = t & 31, warps = threads >> 5;
  if (t < warps * 32)
    for (int g = t >> 5; g < a.n_group; g += warps) {
      float u = 0.f, v = 0.f;
      for (int i = lane; i < k.chunks && k.first + i < a.max_chunks; i += 32) {
        const float *p = a.partial + ((size_t)(k.first + i) * a.n_group + g) * 2;
        u += p[0];
        v += p[1];
      }
      for (int d = 1; d < 32; d <<= 1) u += __shfl_xor_sync(0xffffffffu, u, d), v += __shfl_xor_sync(0xffffffffu, v, d);
      if (lane == 0) {
        const float m = 1.0f / ((float)k.rows * (float)a.t.group_copies[g]);
        sm[2 * g] = u * m;
        sm[2 * g + 1] = v * m;
      }
    }
  __syncthreads();
  GnBack<T, VEC, GATED> back;
  back.setup(a, k, ch, sm + 2 * a.n_group);
  float s1[VEC], s2[VEC];
#pragma unroll
  for (int q = 0; q < VEC; ++q) {
    const int g = a.t.group_of_channel[ch + q];
    s1[q] = a.t.scalar_of_channel[ch + q] >= 0 ? sm[2 * g] : 0.f;
    s2[q] = sm[2 * g + 1];
  }
  for (int row0 = k.lo; row0 < k.hi; row0 += 2 * R) {
    float hat[2][VEC], dz[2][VEC];
    back.rows(a, k, row0, ch, hat, dz);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = row0 + u * R + ty;
      if (row >= k.hi) continue;
#pragma unroll
      for (int q = 0; q < VEC; ++q) dz[u][q] = back.r[q] * (fmaf(dz[u][q], back.w[q], -s1[q]) - hat[u][q] * s2[q]);
      store<T, VEC>(out + (size_t)row * a.c, dz[u]);
    }
  }
}

struct GnShape {
  int vec, tx, ty, chunk_rows, max_chunks;
};

int type_bytes(int type) { return type == SSC_PREC_FP32 ? 4 : 2; }

// Chunks: about four blocks to an SM, at least eight rows to a thread.  (Halves and doubles of this were as fast or slower.)
GnShape gn_shape(int n, int batch, int c, int vec) {
  GnShape s;
  s.vec = vec;
  s.tx = c / vec;
  s.ty = s.tx >= 256 ? 1 : 256 / s.tx;
  const long long unit = 4ll * s.ty, want = ((long long)n + sm_count() * 4 - 1) / (sm_count() * 4);
  long long rows = (want + unit - 1) / unit * unit;
  if (rows < 2 * unit) rows = 2 * unit;
  s.chunk_rows = (int)(rows < 1 << 30 ? rows : 1 << 30);
  s.max_chunks = n / s.chunk_rows + batch + 2;
  return s;
}

int gn_vec(int c, int c_out, int type, const void *x, const void *y, const void *z, int out_type) {
  for (int v = 16 / type_bytes(type); v > 1; v /= 2) {
    if (c % v || c_out % v) continue;
    const uintptr_t in = (uintptr_t)v * type_bytes(type), out = (uintptr_t)v * type_bytes(out_type);
    if (((uintptr_t)x | (uintptr_t)z) % in == 0 && (uintptr_t)y % out == 0) return v;
  }
  return 1;
}

// The partial results for any vector width: one channel a thread makes the most blocks.
size_t gn_scratch(int n, int batch, int c, int n_group, int n_cols) {
  int most = 0;
  for (int v = 1; v <= 8; v *= 2)
    if (c % v == 0 && c / v <= kGnThreads) {
      const GnShape s = gn_shape(n, batch, c, v);
      if (s.max_chunks > most) most = s.max_chunks;
    }
  return (size_t)most * (2 * (size_t)n_group + (size_t)n_cols) * sizeof(float) + 16;
}

int gn_fill(GnArgs &a, const int32_t *table, const char *what) {
  SSC_REQUIRE(a.n >= 0 && a.batch >= 1 && a.c >= 1 && a.c_out >= 1 && a.n_gate >= 0 && a.c_out + a.n_gate == a.c, "%s: bad sizes", what);
  SSC_REQUIRE(a.n_group >= 1 && a.n_group <= a.c && a.n_field >= 1 && a.n_field <= a.c && a.n_scalar >= 0 && a.n_scalar <= a.n_field, "%s: bad layout", what);
  SSC_REQUIRE(a.scalar_act >= 0 && a.scalar_act <= 4 && a.gate_act >= 0 && a.gate_act <= 4, "%s: unknown activation", what);
  SSC_REQUIRE(a.eps > 0.f, "%s: eps must be positive", what);
  SSC_REQUIRE(table && a.offsets && a.stats && (a.n == 0 || (a.x && a.out)), "%s: null pointer", what);
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
  return SSC_OK;
}

template <class T, class TO, int VEC>
cudaError_t gn_fwd(const GnArgs &a, const GnShape &s, cudaStream_t st) {
  const dim3 block(s.tx, s.ty), grid(s.max_chunks);
  const size_t stats = 2 * (size_t)s.ty * a.c * sizeof(float);
  const size_t room = (2 * (size_t)a.n_group + 8 * (size_t)s.ty * a.n_gate) * sizeof(float);
  auto apply = a.n_gate ? gn_apply_kernel<T, TO, VEC, true> : gn_apply_kernel<T, TO, VEC, false>;
  cudaError_t e;
  if (stats > 49152 && (e = allow_smem((const void *)gn_stats_kernel<T, VEC>, stats)) != cudaSuccess) return e;
  if (room > 49152 && (e = allow_smem((const void *)apply, room)) != cudaSuccess) return e;
  if ((e = launch_ready(gn_stats_kernel<T, VEC>, grid, block, stats, st, a)) != cudaSuccess) return e;
  return launch_ready(apply, grid, block, room, st, a);
}

template <class T, int VEC>
cudaError_t gn_bwd(const GnArgs &a, const GnShape &s, cudaStream_t st) {
  const dim3 block(s.tx, s.ty);
  const size_t gates = 2 * (size_t)s.ty * (a.n_gate ? a.n_gate + a.c_out : 0), sums = 2 * (size_t)s.ty * a.c;
  const size_t first = (gates > sums ? gates : sums) * sizeof(float);
  size_t second = 2 * (size_t)a.n_group + gates;
  if (second < (size_t)s.tx * s.ty) second = (size_t)s.tx * s.ty;
  second *= sizeof(float);
  auto one = a.n_gate ? gn_bwd_sums_kernel<T, VEC, true> : gn_bwd_sums_kernel<T, VEC, false>;
  auto two = a.n_gate ? gn_bwd_apply_kernel<T, VEC, true> : gn_bwd_apply_kernel<T, VEC, false>;
  cudaError_t e;
  if (first > 49152 && (e = allow_smem((const void *)one, first)) != cudaSuccess) return e;
  if (second > 49152 && (e = allow_smem((const void *)two, second)) != cudaSuccess) return e;
  const int sum_blocks = ceil_div(a.n_field + a.n_scalar, kGnSum);
  if ((e = launch_ready(one, dim3(s.max_chunks), block, first, st, a)) != cudaSuccess) return e;
  return launch_ready(two, dim3(s.max_chunks + sum_blocks), block, second, st, a, sum_blocks);
}

template <class T, class TO>
cudaError_t gn_fwd_vec(const GnArgs &a, const GnShape &s, cudaStream_t st) {
  switch (s.vec) {
    case 8: if constexpr (sizeof(T) == 2) return gn_fwd<T, TO, 8>(a, s, st);
    case 4: return gn_fwd<T, TO, 4>(a, s, st);
    case 2: return gn_fwd<T, TO, 2>(a, s, st);
    default: return gn_fwd<T, TO, 1>(a, s, st);
  }
}
template <class T>
cudaError_t gn_bwd_vec(const GnArgs &a, const GnShape &s, cudaStream_t st) {
  switch (s.vec) {
    case 8: if constexpr (sizeof(T) == 2) return gn_bwd<T, 8>(a, s, st);
    case 4: return gn_bwd<T, 4>(a, s, st);
    case 2: return gn_bwd<T, 2>(a, s, st);
    default: return gn_bwd<T, 1>(a, s, st);
  }
}
bool known_type(int t) { return t == SSC_PREC_FP32 || t == SSC_PREC_F16 || t == SSC_PREC_BF16; }

}  // namespace
}  // namespace ssc

extern "C" size_t ssc_group_norm_scratch_bytes(int n, int batch, int c, int n_group, int n_field, int n_scalar) {
  if (n < 0 || batch < 1 || c < 1 || n_group < 0 || n_field < 0 || n_scalar < 0) return 0;
  return ssc::gn_scratch(n, batch, c, n_group, n_field + n_scalar);
}

extern "C" int ssc_group_norm_fwd(const void *x, int type, int n, int c, const int32_t *offsets, int batch, const int32_t *table, int n_field,
                                  int n_scalar, int n_group, int n_gate, const float *weight, const float *bias, float eps, int scalar_act, int gate_act,
                                  void *out, int out_type, float *stats, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace ssc;
  SSC_REQUIRE(known_type(type) && known_type(out_type) && (type == out_type || type == SSC_PREC_FP32), "group_norm_fwd: unknown types");
  GnArgs a = {};
  a.x = x; a.out = out; a.n = n; a.c = c; a.c_out = c - n_gate; a.n_gate = n_gate; a.n_group = n_group; a.n_field = n_field; a.n_scalar = n_scalar;
  a.batch = batch; a.offsets = offsets; a.weight = weight; a.bias = bias; a.eps = eps; a.scalar_act = scalar_act; a.gate_act = gate_act; a.stats = stats;
  if (int e = gn_fill(a, table, "group_norm_fwd")) return e;
  if (n == 0) return SSC_OK;
  const GnShape s = gn_shape(n, batch, c, gn_vec(c, a.c_out, type, x, out, x, out_type));
  SSC_REQUIRE(s.tx <= kGnThreads, "group_norm_fwd: %d channels, at most %d of this alignment", c, kGnThreads * s.vec);
  a.chunk_rows = s.chunk_rows;
  a.max_chunks = s.max_chunks;
  if (scratch == nullptr || scratch_bytes < 2 * (size_t)s.max_chunks * n_group * sizeof(float)) return fail(SSC_ERR_SCRATCH, "group_norm_fwd: scratch too small");
  a.partial = (float *)scratch;
  const cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (type == SSC_PREC_F16) e = gn_fwd_vec<__half, __half>(a, s, st);
  else if (type == SSC_PREC_BF16) e = gn_fwd_vec<__nv_bfloat16, __nv_bfloat16>(a, s, st);
  else if (out_type == SSC_PREC_F16) e = gn_fwd_vec<float, __half>(a, s, st);
  else if (out_type == SSC_PREC_BF16) e = gn_fwd_vec<float, __nv_bfloat16>(a, s, st);
  else e = gn_fwd_vec<float, float>(a, s, st);
  if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "group_norm_fwd: %s", cudaGetErrorString(e));
  note_launches(2);
  SSC_CHECK_LAUNCH("group_norm_fwd");
  return SSC_OK;
}

extern "C" int ssc_group_norm_bwd(const void *x, const void *gy, int type, int n, int c, const int32_t *offsets, int batch, const int32_t *table,
                                  int n_field, int n_scalar, int n_group, int n_gate, const float *weight, const float *bias, float eps, int scalar_act,
                                  int gate_act, const float *stats, void *gx, float *d_weight, float *d_bias, void *scratch, size_t scratch_bytes,
                                  void *stream) {
  using namespace ssc;
  SSC_REQUIRE(known_type(type), "group_norm_bwd: unknown type");
  GnArgs a = {};
  a.x = x; a.gy = gy; a.out = gx; a.n = n; a.c = c; a.c_out = c - n_gate; a.n_gate = n_gate; a.n_group = n_group; a.n_field = n_field;
  a.n_scalar = n_scalar; a.batch = batch; a.offsets = offsets; a.weight = weight; a.bias = bias; a.eps = eps; a.scalar_act = scalar_act;
  a.gate_act = gate_act; a.stats = const_cast<float *>(stats); a.d_weight = d_weight; a.d_bias = d_bias;
  if (int e = gn_fill(a, table, "group_norm_bwd")) return e;
  SSC_REQUIRE((n == 0 || gy) && d_weight && (n_scalar == 0 || d_bias), "group_norm_bwd: null pointer");
  const cudaStream_t st = as_stream(stream);
  if (n == 0) {
    cudaError_t e = cudaMemsetAsync(d_weight, 0, n_field * sizeof(float), st);
    if (e == cudaSuccess && n_scalar) e = cudaMemsetAsync(d_bias, 0, n_scalar * sizeof(float), st);
    if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "group_norm_bwd: %s", cudaGetErrorString(e));
    return SSC_OK;
  }
  const GnShape s = gn_shape(n, batch, c, gn_vec(c, a.c_out, type, x, gx, gy, type));
  SSC_REQUIRE(s.tx <= kGnThreads, "group_norm_bwd: %d channels, at most %d of this alignment", c, kGnThreads * s.vec);
  a.chunk_rows = s.chunk_rows;
  a.max_chunks = s.max_chunks;
  if (scratch == nullptr || scratch_bytes < (size_t)s.max_chunks * (2 * (size_t)n_group + n_field + n_scalar) * sizeof(float))
    return fail(SSC_ERR_SCRATCH, "group_norm_bwd: scratch too small");
  a.partial = (float *)scratch;
  a.fields = a.partial + 2 * (size_t)s.max_chunks * n_group;
  cudaError_t e = type == SSC_PREC_F16 ? gn_bwd_vec<__half>(a, s, st) : type == SSC_PREC_BF16 ? gn_bwd_vec<__nv_bfloat16>(a, s, st) : gn_bwd_vec<float>(a, s, st);
  if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "group_norm_bwd: %s", cudaGetErrorString(e));
  note_launches(2);
  SSC_CHECK_LAUNCH("group_norm_bwd");
  return SSC_OK;
}
