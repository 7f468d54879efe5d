// Gated feed-forward of rows: y = (act(x Wg' + bg) * (x Wu' + bu)) Wo' + bo (+ residual), and its gradients.
//
// Forward: one product for gate and up, whose epilogue applies the activation and multiplies (h leaves the SM once, in
// the rows' type), one product for the way out.  Backward: gate and up are computed again together with dh = dy Wo, and the epilogue
// turns the three into h, dg = dh u act'(g) and du = dh act(g) (keeping g and u would cost more memory traffic than their products
// cost time up to 700 channels, and two roundings); then dx = dg Wg + du Wu, dWin = [dg, du]' x and dWo = dy' h, whose long sums
// are split over the rows and added in a fixed order.
//
// All of them are one kernel: pairs of CTAs with tiles of 256 rows in tensor memory, half of each operand in either CTA, operands by TMA, a warp
// that issues the products and others that empty the accumulators, two of which are in turn.  Operands are 16-bit; float32 rows are the sum of
// three bfloat16 planes (24 bits), and a product the sum of the six products of planes that reach 2^-24, the small ones first.
// Of 16-bit rows h, dg and du are rounded to 16 bits as well, as the operands they become: a second plane of each would double the products behind it and
// what leaves the SM, which bounds them already.  Errors are 0.0024 (bf16) and 2.9e-4 (fp16) of a result that way, where
// the rounding of the result alone is 0.0017 and 2.1e-4.  Few rows on plain lanes keep h in float32.
//
// 65536 rows 256 -> 1024 -> 256 in bf16, forward 126 us, backward 311 (rates of a cool GPU; under its power limit 500 for both): gate, up and h
// 77 (893 TFLOP/s of its two products, bound by the way out: 134 MB of h through shared memory), the way out 49, h, dg and du 140 (403 MB), dx 68, the
// gradients of Win and Wo 56 and 37, their sums 10.  float32, 16384 rows 128 -> 512 -> 128, 268 us for both: h, dg and du 68, nine planes whose splitting and stores
// bound it.  One row 256 -> 1024 -> 256 3.7 us, two launches and two latencies.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ssc_common.cuh"
#include "ssc_rows_act.cuh"
#include "ssc_tc_ptx.cuh"

namespace ssc {
namespace {

enum Epilogue { kGate, kBack, kRows, kPart };
constexpr int kBox = 64;                      // TMA boxes: 64 x 64 elements, 128-byte rows
constexpr uint32_t kBoxBytes = kBox * kBox * 2;
constexpr int kTileM = 256;                   // of a pair of CTAs, half of it each
constexpr uint32_t kStageBytes = 4 * kBoxBytes;     // two boxes of A, up to two of B
template <int EPI>
constexpr int kStages = EPI == kBack ? 4 : 5;
template <int EPI>
constexpr uint32_t kOutBytes = EPI == kBack ? 98304 : 65536;      // rows on their way out, a share for each of the warps that empty accumulators
// Warps: TMA, products, tensor memory, an idle one, then those for the accumulators: sixteen, eight where sums in registers (LONG) need the room.
template <bool LONG>
constexpr int kSides = LONG ? 2 : 4;                        // shares of a tile's columns
template <bool LONG>
constexpr int kThreads = 128 + 128 * kSides<LONG>;
template <int EPI>
constexpr uint32_t kSmemBytes = kStages<EPI> * kStageBytes + kOutBytes<EPI> + 1024;

enum Half { kNone, kByK, kByBox, kByM };      // what chooses between the two matrices of an operand (gate and up)

struct Segment {
  int a_mn, b_mn;            // 1: stored with the rows of the product (not the summed index) contiguous
  int a_half, b_half;
  int a_planes, b_planes;    // matrices of one plane: 1 or 2
  int blocks;                // of 64 along the summed index
  int half_blocks;           // kByK: blocks of the first matrix
  uint32_t idesc;            // of the product: types, which operand lies which way round, 256 rows and the columns
  int boxes_b;               // of each CTA: half of the product's columns (kByBox: of one matrix in each)
};
struct FfMaps {
  CUtensorMap a[2], b[2];
  CUtensorMap out[2];        // of out and out2, where rows can be stored by boxes
};
struct FfParams {
  Segment seg[2];
  int n_seg, pairs;
  int tiles_m, tiles_n, splits, m_half;        // tiles; m_half: tiles of the first matrix (kByM)
  int step_n;                                  // columns of the result to a tile
  int rows, cols;                              // of the result (one matrix)
  int act;
  const void *bias;                            // of the result's columns; kGate / kBack: [2][hidden]
  const void *residual;                        // kRows: rows of T; kBack of float32: dh [rows][pitch]
  void *out, *out2;                            // kGate: h; kBack: h, dg|du; kRows: result; kPart: float [splits][rows of all][cols]
  int pitch;                                   // of out
  size_t plane;                                // kPart: elements of a share
  int boxes;                                   // out (and out2) are stored by boxes (maps.out), else from registers
  int vec;                                     // rows of the residual are aligned to 16 bytes
  int accumulate;                              // kPart: add to what is there
  int32_t *status, *alarm;
};

// A box into this CTA's shared memory; its bytes count on a barrier of either CTA.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void arrive_there(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

// Operands of a stage: rows of 128 bytes, 128-byte swizzle.  Summed index contiguous: groups of eight rows 1024 bytes
// apart, 32 bytes a step of 16.  Rows contiguous: blocks of 64 rows a box apart, eight steps of the summed index 1024 bytes.
__device__ __forceinline__ uint32_t operand_lo(uint32_t addr, int mn) { return ((addr >> 4) & 0x3FFFu) | (mn ? (kBoxBytes >> 4) << 16 : 1u << 16); }

__constant__ const int8_t kPlaneA[6] = {2, 0, 1, 1, 0, 0}, kPlaneB[6] = {0, 2, 1, 0, 1, 0};

template <class T>
__device__ __forceinline__ void add16(float *v, const T *p, int left, int vec) {
  if (vec && left >= 16) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16; i += N) {
      struct alignas(16) { T v[N]; } k;
      *(int4 *)&k = *(const int4 *)(p + i);
#pragma unroll
      for (int q = 0; q < N; ++q) v[i + q] += (float)k.v[q];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) v[i] += (float)p[i];
  }
}
// The next of three bfloat16 planes of v, a word to two values; v keeps what is left.  What is not finite is in the first plane alone.
template <int N, bool FIRST>
__device__ __forceinline__ void next_plane(float *v, uint32_t *w) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const __nv_bfloat162 k = __floats2bfloat162_rn(v[i], v[i + 1]);
    w[i / 2] = *(const uint32_t *)&k;
    const float a = __uint_as_float(w[i / 2] << 16), b = __uint_as_float(w[i / 2] & 0xFFFF0000u);
    const float2 left = halves(fma_pair(pair_of(a, b), pair_of(-1.f, -1.f), pair_of(v[i], v[i + 1])));
    v[i] = !FIRST || fabsf(a) < INFINITY ? left.x : 0.f;
    v[i + 1] = !FIRST || fabsf(b) < INFINITY ? left.y : 0.f;
  }
}
template <int N>
__device__ __forceinline__ void next_plane(float *v, uint32_t *w, int plane) {
  if (plane == 0) next_plane<N, true>(v, w);
  else next_plane<N, false>(v, w);
}

// A warp's way out of 32 rows of up to 32 columns: each lane puts its row's 16 columns into the warp's shared memory, one lane sends the box off.  Rows
// from registers cost as much time as the products did (131072 rows 512 -> 2048 in bf16: 549 us, 394 without them).
// Boxes of 32 columns: rows of 64 bytes (16-bit) or 128 (float32), or of 16 columns, 32 bytes; swizzled as the copy engine has it, which
// keeps lanes on different banks.  (kBack of float32 rows, 16384 of 128 -> 512: 65 us; by boxes of 32 columns, which leave registers for half of the warps, 70.)
struct Outbox {
  uint32_t at;             // the warp's shared memory: slots taken in turn
  uint32_t slot, slots, slot_bytes;
  __device__ __forceinline__ void open(uint32_t where, uint32_t size, uint32_t each) {
    at = where;
    slot_bytes = each;
    slots = size / each;
    slot = 0;
  }
  // Room for one more box (the whole warp): what was sent last may still be read, the slots before it not.
  __device__ __forceinline__ uint32_t room() {
    if ((threadIdx.x & 31) == 0) {
      if (slots == 1) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      else if (slots < 4) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      else asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory");
    }
    __syncwarp();
    const uint32_t here = at + slot * slot_bytes;
    if (++slot == slots) slot = 0;
    return here;
  }
  // 16 columns (part 0, 1 ... of the box) of the lane's row, as words or as values to be rounded.
  template <int ROW_BYTES, int BYTES>
  __device__ __forceinline__ void put_words(uint32_t box, int part, const uint32_t *w) {
    const uint32_t lane = threadIdx.x & 31;
    constexpr uint32_t mask = ROW_BYTES / 16 - 1;
    const uint32_t row = box + lane * ROW_BYTES, turn = lane / (128 / ROW_BYTES) & mask;
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint32_t to = row + (((uint32_t)(part * (BYTES / 16) + i) ^ turn) << 4);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3]) : "memory");
    }
  }
  template <class V, int COLS = 32>
  __device__ __forceinline__ void put(uint32_t box, int part, const float *v) {
    struct alignas(16) { V v[16]; } k;
#pragma unroll
    for (int q = 0; q < 16; ++q) k.v[q] = (V)v[q];
    put_words<COLS * sizeof(V), 16 * sizeof(V)>(box, part, (const uint32_t *)&k);
  }
  // One value of a box of 32 float32 columns.
  static __device__ __forceinline__ float get(uint32_t box, uint32_t row, uint32_t col) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(box + row * 128 + ((((col >> 2) ^ row) & 7) << 4) + (col & 3) * 4) : "memory");
    return v;
  }
  __device__ __forceinline__ void send(uint32_t box, const CUtensorMap *map, int x, int y, int z) {
    fence_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(box) : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  __device__ __forceinline__ void close() {
    if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
};
__device__ __forceinline__ void tmem_floats(float *v, uint32_t addr) { tmem_ld16((uint32_t *)v, addr); }
__device__ __forceinline__ void tmem_arrived() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The tiles of a pair of CTAs, stepped through without a division: the roles that walk are single warps, whose every instruction is
// waited for (with divisions for tiles and shares, products of K = 256 spent half of their time between tiles).
struct Walk {
  int n, m, split;      // column tile, row tile, share
  int dn, dm, ds;
  __device__ __forceinline__ explicit Walk(const FfParams &p) {
    const int t = blockIdx.x >> 1, by = gridDim.x >> 1;
    split_up(p, t, n, m, split);
    split_up(p, by, dn, dm, ds);
  }
  static __device__ __forceinline__ void split_up(const FfParams &p, int t, int &n, int &m, int &split) {
    n = t % p.tiles_n;
    t /= p.tiles_n;
    m = t % p.tiles_m;
    split = t / p.tiles_m;
  }
  __device__ __forceinline__ bool more(const FfParams &p) const { return split < p.splits; }
  __device__ __forceinline__ void next(const FfParams &p) {
    n += dn;
    m += dm;
    split += ds;
    if (n >= p.tiles_n) n -= p.tiles_n, ++m;
    if (m >= p.tiles_m) m -= p.tiles_m, ++split;
  }
};
// The blocks of 64 of a segment's sum in a share.
__device__ __forceinline__ void share_of_sum(const FfParams &p, int g, int split, int &first, int &blocks) {
  first = 0;
  blocks = p.seg[g].blocks;
  if (p.splits > 1) {
    first = (int)((uint32_t)blocks * (uint32_t)split / (uint32_t)p.splits);
    blocks = (int)((uint32_t)blocks * (uint32_t)(split + 1) / (uint32_t)p.splits) - first;
  }
}

// The steps of a tile's sum: `blocks` of 64 for each pair of planes.  Tensor memory's additions cut off instead of rounding, which
// adds up (1.5e-6 of gx over 1024 terms): float32 results leave tensor memory after every kLeave blocks of the last
// pair, the largest one, and are added up in registers.  16-bit results stay.
constexpr int kLeave = 4;
__device__ __forceinline__ int part_count(int blocks, int pairs) { return pairs == 1 || blocks <= kLeave ? 1 : (blocks + kLeave - 1) / kLeave; }
__device__ __forceinline__ int part_begin(int blocks, int pairs, int part) {
  return part == 0 ? 0 : min((pairs - 1) * blocks + part * (pairs == 1 ? blocks : kLeave), pairs * blocks);
}

__device__ __forceinline__ int parts_of(const FfParams &p, int split) {
  if (p.pairs == 1) return 1;
  int most = 1;
  for (int g = 0; g < p.n_seg; ++g) {
    int first, blocks;
    share_of_sum(p, g, split, first, blocks);
    most = max(most, part_count(blocks, p.pairs));
  }
  return most;
}

// dh of float32 rows, which has been multiplied before.
__device__ __forceinline__ void stored_dh(const FfParams &p, int row, int n, float *d) {
#pragma unroll
  for (int i = 0; i < 16; ++i) d[i] = 0.f;
  if (row < p.rows && n < p.cols) add16<float>(d, (const float *)p.residual + (size_t)row * p.pitch + n, p.cols - n, 1);
}

// A plane of 32 columns of hidden rows (16-bit, or one of the three of float32 rows) goes out as a box.
template <class T>
__device__ __forceinline__ void send_hidden(Outbox &box, const CUtensorMap *map, float (*v)[16], int n, int row0, int z, int planes_apart) {
  if (sizeof(T) == 2) {
    const uint32_t at = box.room();
    box.put<T>(at, 0, v[0]);
    box.put<T>(at, 1, v[1]);
    box.send(at, map, n, row0, z);
  } else {
#pragma unroll
    for (int plane = 0; plane < 3; ++plane) {
      const uint32_t at = box.room();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[8];
        next_plane<16>(v[h], w, plane);
        box.put_words<64, 32>(at, h, w);
      }
      box.send(at, map, n, row0, z + plane * planes_apart);
    }
  }
}

// 16 columns (half `half` of a box) of a warp's rows, row0 the first of them: gate v, up u, dh d.
template <class T>
__device__ __forceinline__ void finish_back(const FfParams &p, const FfMaps &maps, Outbox &box, int row0, int n, int half, float *v, float *u, float *d) {
  const int left = p.cols - n;
  if (p.bias && left > 0) {
    add16<T>(v, (const T *)p.bias + n, left, 0);
    add16<T>(u, (const T *)p.bias + p.cols + n, left, 0);
  }
  float s[16], h[16];
  act_slopes<sizeof(T) == 4, 16>(v, s, p.act);
#pragma unroll
  for (int i = 0; i < 16; ++i) h[i] = v[i];
  multiply<16>(h, h, u);        // act(g) u
  multiply<16>(u, u, s);
  multiply<16>(u, u, d);        // dh u act'(g)
  multiply<16>(v, v, d);        // dh act(g)
  if constexpr (sizeof(T) == 2) {
    if (half == 0) {            // three boxes at a time
      if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
    }
    box.put<T>(box.at, half, h);
    box.put<T>(box.at + 2048, half, u);
    box.put<T>(box.at + 4096, half, v);
    if (half == 1) {
      box.send(box.at, &maps.out[0], n - 16, row0, 0);
      box.send(box.at + 2048, &maps.out[1], n - 16, row0, 0);
      box.send(box.at + 4096, &maps.out[1], n - 16, row0, 1);
    }
  } else if (left > 0) {
#pragma unroll
    for (int o = 0; o < 3; ++o) {
      float *from = o == 0 ? h : o == 1 ? u : v;
#pragma unroll
      for (int plane = 0; plane < 3; ++plane) {
        uint32_t w[8];
        next_plane<16>(from, w, plane);
        const uint32_t at = box.room();
        box.put_words<32, 32>(at, 0, w);
        box.send(at, o == 0 ? &maps.out[0] : &maps.out[1], n, row0, o == 0 ? plane : 2 * plane + o - 1);
      }
    }
  }
}

// 32 columns from column n on of a warp's rows of the result, two times 16: v (kGate: gate, u: up).
template <int EPI, class T>
__device__ __forceinline__ void finish(const FfParams &p, const FfMaps &maps, Outbox &box, int split, int half_m, int row0, int n, float (*v)[16], float (*u)[16]) {
  const int row = row0 + (threadIdx.x & 31);
  if (EPI == kGate) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int left = p.cols - n - 16 * q;
      if (p.bias && left > 0) {
        add16<T>(v[q], (const T *)p.bias + n + 16 * q, left, 0);
        add16<T>(u[q], (const T *)p.bias + p.cols + n + 16 * q, left, 0);
      }
      act_values<sizeof(T) == 4, 16>(v[q], p.act);
      multiply<16>(v[q], v[q], u[q]);
    }
    send_hidden<T>(box, &maps.out[0], v, n, row0, 0, 1);
    return;
  }
  using V = std::conditional_t<EPI == kPart, float, T>;
  if (p.boxes) {
    if (EPI == kRows) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int left = p.cols - n - 16 * q;
        if (left <= 0) continue;
        if (p.bias) add16<T>(v[q], (const T *)p.bias + n + 16 * q, left, 0);
        if (p.residual && row < p.rows) add16<T>(v[q], (const T *)p.residual + (size_t)row * p.pitch + n + 16 * q, left, p.vec);
      }
    }
    const uint32_t at = box.room();
    box.put<V>(at, 0, v[0]);
    box.put<V>(at, 1, v[1]);
    box.send(at, &maps.out[0], n, row0, EPI == kPart ? split * (p.m_half < p.tiles_m ? 2 : 1) + half_m : 0);
  } else {
    // a lane to a column: rows that are no multiple of 16 bytes, one value at a time
    const uint32_t lane = threadIdx.x & 31;
    box.put<float>(box.at, 0, v[0]);
    box.put<float>(box.at, 1, v[1]);
    __syncwarp();
    const int col = n + (int)lane, many = min(32, p.rows - row0);
    if (col < p.cols) {
      const float bias = EPI == kRows && p.bias ? (float)((const T *)p.bias)[col] : 0.f;
      V *o = (V *)p.out + (EPI == kPart ? (size_t)split * p.plane : 0) + ((size_t)half_m * p.rows + row0) * p.pitch + col;
      const T *add = EPI == kRows && p.residual ? (const T *)p.residual + (size_t)row0 * p.pitch + col : nullptr;
#pragma unroll 8
      for (int r = 0; r < many; ++r) {
        float x = Outbox::get(box.at, r, lane) + bias;
        if (add) x += (float)add[(size_t)r * p.pitch];
        if (EPI == kPart && p.accumulate) x += (float)o[(size_t)r * p.pitch];
        o[(size_t)r * p.pitch] = (V)x;
      }
    }
    __syncwarp();
  }
}

// LONG: float32 sums that leave tensor memory in between (part_count).
template <int EPI, class T, bool LONG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads<LONG>, 1) ff_gemm_kernel(const __grid_constant__ FfMaps maps, const FfParams p) {
  after_previous();
  extern __shared__ uint8_t raw[];
  __shared__ alignas(8) uint64_t bars[2 * kStages<EPI> + 5];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;
  const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages<EPI>, acc_full = empty + 8 * kStages<EPI>, acc_empty = acc_full + 16, done = acc_empty + 16;
  const int warp = warp_id(), rank = blockIdx.x & 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages<EPI>; ++s) {
      mbar_init(full + 8 * s, 1);                       // the first CTA's: both CTAs' boxes count there
      mbar_init(empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + 8 * b, 1);
      mbar_init(acc_empty + 8 * b, 8 * kSides<LONG>);   // the first CTA's: both CTAs' warps
    }
    mbar_init(done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                       // the other CTA's barriers stand
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  // Accumulators: two of 256 columns in turn.  kBack with three products: gate and up in the first 256 columns, dh in the others, in turn, so that
  // the next tile's dh is multiplied while this tile's values are taken out.
  constexpr bool kThree = EPI == kBack && sizeof(T) == 2;

  if (warp == 0) {
    // operands
    const uint32_t full_there = peer_address(full, 0);
    uint32_t slot = 0, phase = 1, step = 0;
    bool ok = true;
    for (Walk k(p); k.more(p) && ok; k.next(p)) {
      const int half_m = k.m >= p.m_half ? 1 : 0, m0 = (k.m - half_m * p.m_half) * kTileM + rank * (kTileM / 2);
      const int parts = parts_of(p, k.split);
      for (int part = 0; part < parts; ++part)
        for (int g = 0; g < p.n_seg; ++g) {
          const Segment &s = p.seg[g];
          int kb0, blocks;
          share_of_sum(p, g, k.split, kb0, blocks);
          if (part >= part_count(blocks, p.pairs)) continue;
          const int n0 = k.n * p.step_n + (s.b_half == kByBox ? 0 : rank * s.boxes_b * kBox), end = part_begin(blocks, p.pairs, part + 1);
          const CUtensorMap *map_a = &maps.a[g], *map_b = &maps.b[g];
          const uint32_t bytes = 2 * (2 + s.boxes_b) * kBoxBytes;
          int pair = part == 0 ? 0 : p.pairs - 1, i = part_begin(blocks, p.pairs, part), kb = i - pair * blocks;
          while (i < end && ok) {
            // a run of blocks of one pair of planes in one matrix
            const int by_k = kb0 + kb >= s.half_blocks ? 1 : 0;
            const int run = min(min(end - i, blocks - kb), by_k ? 1 << 30 : s.half_blocks - kb0 - kb);
            const int pa = p.pairs == 1 ? 0 : kPlaneA[pair], pb = p.pairs == 1 ? 0 : kPlaneB[pair];
            const int za = pa * s.a_planes + (s.a_half == kByK ? by_k : s.a_half == kByM ? half_m : 0);
            const int zb = pb * s.b_planes + (s.b_half == kByK ? by_k : s.b_half == kByBox ? rank : 0);
            int kk = (kb0 + kb - by_k * s.half_blocks) * kBox;
            for (int j = 0; j < run && ok; ++j, kk += kBox, ++step) {
              ok = mbar_wait_straight(empty + 8 * slot, phase, &abort_flag);
              const uint32_t at = ring + slot * kStageBytes, bar = full_there + 8 * slot;
              if (ok && elect_one()) {
                if (rank == 0) mbar_expect_tx(full + 8 * slot, bytes);
                if (s.a_mn) {
                  tma_box(at, map_a, m0, kk, za, bar);
                  tma_box(at + kBoxBytes, map_a, m0 + kBox, kk, za, bar);
                } else {
                  tma_box(at, map_a, kk, m0, za, bar);
                  tma_box(at + kBoxBytes, map_a, kk, m0 + kBox, za, bar);
                }
                if (s.b_mn) {
                  tma_box(at + 2 * kBoxBytes, map_b, n0, kk, zb, bar);
                  if (s.boxes_b == 2) tma_box(at + 3 * kBoxBytes, map_b, n0 + kBox, kk, zb, bar);
                } else {
                  tma_box(at + 2 * kBoxBytes, map_b, kk, n0, zb, bar);
                  if (s.boxes_b == 2) tma_box(at + 3 * kBoxBytes, map_b, kk, n0 + kBox, zb, bar);
                }
              }
              if (++slot == kStages<EPI>) slot = 0, phase ^= 1;
            }
            i += run;
            kb += run;
            if (kb == blocks) kb = 0, ++pair;
          }
        }
    }
    if (abort_flag && rank == 0)      // copies in flight, the other CTA's too, arrive before the blocks leave
      for (uint32_t s = step > kStages<EPI> ? step - kStages<EPI> : 0; s < step; ++s) mbar_wait_drain(full + 8 * (s % kStages<EPI>), (s / kStages<EPI>) & 1);
  } else if (warp == 1 && rank == 0) {
    // products
    uint32_t slot = 0, phase = 0, turn = 0;
    bool ok = true;
    for (Walk k(p); k.more(p) && ok; k.next(p)) {
      const int parts = parts_of(p, k.split);
      for (int part = 0; part < parts && ok; ++part, ++turn) {
        const uint32_t buf = turn & 1;
        ok = mbar_wait_straight_cluster(acc_empty + 8 * buf, ((turn >> 1) & 1) ^ 1, &abort_flag);
        tc_fence_after();
        for (int g = 0; g < p.n_seg; ++g) {
          const Segment &s = p.seg[g];
          int first, blocks;
          share_of_sum(p, g, k.split, first, blocks);
          if (part >= part_count(blocks, p.pairs)) continue;
          if (kThree && g == 1 && turn > 0) {           // gate and up of the tile before have been taken out
            ok = ok && mbar_wait_straight_cluster(acc_empty + 8 * (buf ^ 1), ((turn - 1) >> 1) & 1, &abort_flag);
            tc_fence_after();
          }
          const int steps = part_begin(blocks, p.pairs, part + 1) - part_begin(blocks, p.pairs, part);
          const uint32_t idesc = s.idesc, d = tmem + (kThree ? (g == 0 ? 256 + buf * 128 : 0) : buf * 256), ua = s.a_mn ? 128 : 2, ub = s.b_mn ? 128 : 2;
          const uint32_t a0 = operand_lo(ring, s.a_mn), b0 = operand_lo(ring + 2 * kBoxBytes, s.b_mn);
          for (int i = 0; i < steps && ok; ++i) {
            ok = mbar_wait_straight_cluster(full + 8 * slot, phase, &abort_flag);
            tc_fence_after();
            const uint32_t a = a0 + slot * (kStageBytes >> 4), b = b0 + slot * (kStageBytes >> 4);
            if (ok && elect_one()) {
#pragma unroll
              for (uint32_t q = 0; q < 4; ++q) mma_pair<true>(d, a + q * ua, b + q * ub, idesc, (i | (int)q) != 0 ? 1u : 0u);
              mma_commit_pair(empty + 8 * slot);
            }
            if (++slot == kStages<EPI>) slot = 0, phase ^= 1;
          }
        }
        if (ok && elect_one()) mma_commit_pair(acc_full + 8 * buf);
      }
    }
  } else if (warp >= 4) {
    // accumulators: a thread has a row and a share of a tile's columns, kGroups times 32 of them from kSets products
    constexpr int kSets = EPI == kGate ? 2 : kThree ? 3 : EPI == kBack ? 2 : 1, kGroups = kSets == 2 ? 2 : 4;      // of 32
    const int quad = warp & 3, side = (warp - 4) >> 2, lane = threadIdx.x & 31;
    const uint32_t lanes = (uint32_t)(32 * quad) << 16, empty_there = peer_address(acc_empty, 0);
    constexpr uint32_t kShare = kOutBytes<EPI> / (4 * kSides<LONG>);
    Outbox box;
    box.open(ring + kStages<EPI> * kStageBytes + (warp - 4) * kShare, kShare, EPI == kBack && sizeof(T) == 4 ? 1024 : EPI == kPart || (EPI == kRows && sizeof(T) == 4) ? 4096 : 2048);
    uint32_t turn = 0;
    bool ok = true;
    for (Walk k(p); k.more(p) && ok; k.next(p)) {
      const int half_m = k.m >= p.m_half ? 1 : 0, m0 = (k.m - half_m * p.m_half) * kTileM + rank * (kTileM / 2), n0 = k.n * p.step_n;
      const int row0 = m0 + 32 * quad, each = p.step_n / kSides<LONG>;
      int first, blocks;
      share_of_sum(p, 0, k.split, first, blocks);
      if constexpr (LONG) {
        float sum[kSets][kGroups][2][16];
#pragma unroll
        for (int i = 0; i < kSets * kGroups * 32; ++i) (&sum[0][0][0][0])[i] = 0.f;
        const int parts = parts_of(p, k.split);
        for (int part = 0; part < parts && ok; ++part, ++turn) {
          const uint32_t buf = turn & 1, acc = tmem + buf * 256 + lanes;
          ok = mbar_wait_uniform(acc_full + 8 * buf, (turn >> 1) & 1, &abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (blocks > 0) {                             // (else an empty share)
#pragma unroll
            for (int s = 0; s < kSets; ++s)
#pragma unroll
              for (int g = 0; g < 2 * kGroups; ++g)
                if (16 * g < each) {
                  float v[16];
                  tmem_floats(v, acc + s * p.step_n + side * each + 16 * g);
                  tmem_arrived();
#pragma unroll
                  for (int i = 0; i < 16; ++i) sum[s][g / 2][g % 2][i] += v[i];
                }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_there(empty_there + 8 * buf);
        }
        if (!ok) break;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int n = n0 + side * each + 32 * g;
          if (32 * g < each && n < p.cols) {
            if constexpr (EPI == kBack) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                float d[16];
                stored_dh(p, row0 + lane, n + 16 * q, d);
                finish_back<T>(p, maps, box, row0, n + 16 * q, q, sum[0][g][q], sum[1][g][q], d);
              }
            } else {
              finish<EPI, T>(p, maps, box, k.split, half_m, row0, n, sum[0][g], sum[kSets > 1 ? 1 : 0][g]);
            }
          }
        }
      } else {
        const uint32_t buf = turn & 1, acc = tmem + (kThree ? 0 : buf * 256) + lanes;
        ok = mbar_wait_uniform(acc_full + 8 * buf, (turn >> 1) & 1, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        for (int c = side * each; c < (side + 1) * each; c += 32) {
          const int n = n0 + c;
          if (n >= p.cols) break;
          const bool last = c + 32 >= (side + 1) * each || n + 32 >= p.cols;      // behind it the accumulator is free
          if constexpr (EPI == kBack) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float v[3][16];
#pragma unroll
              for (int s = 0; s < kSets; ++s) tmem_floats(v[s], (s == 2 ? tmem + 256 + buf * 128 + lanes : acc + s * p.step_n) + c + 16 * q);
              tmem_arrived();
              if (q == 1 && last) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_there(empty_there + 8 * buf);
              }
              if (!kThree) stored_dh(p, row0 + lane, n + 16 * q, v[2]);
              finish_back<T>(p, maps, box, row0, n + 16 * q, q, v[0], v[1], v[2]);
            }
          } else {
            float v[kSets][2][16];
#pragma unroll
            for (int s = 0; s < kSets; ++s)
#pragma unroll
              for (int q = 0; q < 2; ++q) tmem_floats(v[s][q], acc + s * p.step_n + c + 16 * q);
            tmem_arrived();
            if (last) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) arrive_there(empty_there + 8 * buf);
            }
            if (EPI == kPart && blocks == 0) {
#pragma unroll
              for (int i = 0; i < 32; ++i) (&v[0][0][0])[i] = 0.f;      // (an empty share)
            }
            finish<EPI, T>(p, maps, box, k.split, half_m, row0, n, v[0], v[kSets > 1 ? 1 : 0]);
          }
        }
        if (n0 + side * each >= p.cols) {                             // (no columns here)
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_there(empty_there + 8 * buf);
        }
        ++turn;
      }
    }
    box.close();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (abort_flag) {
    if (warp == 1 && rank == 0) {      // products that are still running end before tensor memory is given back
      if (elect_one()) mma_commit_pair(done);
      __syncwarp();
      mbar_wait_drain(done, 0);
    }
    if (threadIdx.x == 0) report_expired(p.status, p.alarm);
  }
  cluster_sync();                                       // neither leaves while the other may still signal it
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  cluster_sync();
}

// Gate and up of rows that are narrow enough to stay in shared memory: a pair of CTAs keeps its 256 rows of x and goes through the hidden columns,
// 64 at a time, with the weights alone coming by.  That halves what is fetched from L2, and accumulators of 128 columns leave room for four
// in turn with a group of warps for each, so that products, special functions and stores of different tiles run side by side.  65536 rows 256 -> 1024
// in bf16: by tiles of 128 hidden columns with rows fetched for each 104 us.  (All sixteen warps on one tile after the other wait for one chain of
// instructions, 117 us; rows of 32 bytes on their way out keep the copy engine busy, 86; dh as a third product leaves room for neither four
// accumulators nor wide boxes, 180 instead of 169.)
struct HiddenParams {
  int rows, cols;                  // cols: hidden
  int blocks;                      // of 64 along c
  int pairs;                       // of planes: 1 or 6
  int tiles_m, tiles_n, chunks;    // 256 rows; 64 columns; shares of the columns a pair goes through with one set of rows
  int act, stages;
  const void *bias;
  uint32_t idesc;
  int32_t *status, *alarm;
};
struct HiddenMaps {
  CUtensorMap x, w_in, h;          // h: boxes of 64 columns (32: planes)
};
constexpr int kKeep = 6;           // blocks of 128 x 64 that stay, at most; the ring needs the rest
constexpr uint32_t kBlockBytes = 2 * kBoxBytes;
// A step brings two blocks of Win': what the two warps that issue do around a step costs as much as the products of one block.
constexpr uint32_t kStepBytes = 2 * kBoxBytes;
constexpr int kHiddenStages = 6;   // at most
constexpr uint32_t kHiddenOut = 65536, kHiddenRoom = 230400;
constexpr int kHiddenThreads = 640;
// Pairs of planes (kPlaneA): the last one that a plane of A is in.
__constant__ const int8_t kLastPair[3] = {5, 3, 0};

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kHiddenThreads, 1) ff_hidden_kernel(const __grid_constant__ HiddenMaps maps, const HiddenParams p) {
  after_previous();
  constexpr int kBufs = 4, kBufCols = 128;
  extern __shared__ uint8_t raw[];
  __shared__ alignas(8) uint64_t bars[2 * kHiddenStages + 2 * kKeep + 2 * kBufs + 1];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;
  const uint32_t outs = (smem_u32(raw) + 1023u) & ~1023u, keep = outs + kHiddenOut, ring = keep + p.blocks * (p.pairs == 1 ? 1 : 3) * kBlockBytes;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kHiddenStages, kept = empty + 8 * kHiddenStages, free_ = kept + 8 * kKeep, acc_full = free_ + 8 * kKeep,
                 acc_empty = acc_full + 8 * kBufs, done = acc_empty + 8 * kBufs;
  const int warp = warp_id(), rank = blockIdx.x & 1, units = p.tiles_m * p.chunks, stride = gridDim.x >> 1, S = p.stages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kHiddenStages + 2 * kKeep + kBufs; ++i) mbar_init(full + 8 * i, 1);
    for (int b = 0; b < kBufs; ++b) mbar_init(acc_empty + 8 * b, 8);      // (the first CTA's: both CTAs' warps)
    mbar_init(done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp == 0) {
    // operands: a block of rows comes with the step that needs it first
    const uint32_t full_there = peer_address(full, 0), kept_there = peer_address(kept, 0);
    int slot = 0, step = 0;
    uint32_t phase = 1, unit = 0;
    bool ok = true;
    for (int u = blockIdx.x >> 1; u < units && ok; u += stride, ++unit) {
      const int m = u / p.chunks, c = u - m * p.chunks, m0 = m * kTileM + rank * (kTileM / 2);
      const int n_begin = c * p.tiles_n / p.chunks, n_end = (c + 1) * p.tiles_n / p.chunks;
      for (int n = n_begin; n < n_end && ok; ++n)
        for (int pair = 0; pair < p.pairs && ok; ++pair) {
          const int pa = p.pairs == 1 ? 0 : kPlaneA[pair], pb = p.pairs == 1 ? 0 : kPlaneB[pair];
          const bool fetch = n == n_begin && pair < 3;
          for (int kb = 0; kb < p.blocks && ok; kb += 2, ++step) {
            const int many = min(2, p.blocks - kb);
            if (fetch)
              for (int j = 0; j < many; ++j) {
                const int at = pa * p.blocks + kb + j;
                ok = ok && mbar_wait_straight(free_ + 8 * at, (unit & 1) ^ 1, &abort_flag);
                if (ok && elect_one()) {
                  if (rank == 0) mbar_expect_tx(kept + 8 * at, 2 * kBlockBytes);
                  tma_box(keep + at * kBlockBytes, &maps.x, (kb + j) * kBox, m0, pa, kept_there + 8 * at);
                  tma_box(keep + at * kBlockBytes + kBoxBytes, &maps.x, (kb + j) * kBox, m0 + kBox, pa, kept_there + 8 * at);
                }
              }
            ok = ok && mbar_wait_straight(empty + 8 * slot, phase, &abort_flag);
            if (ok && elect_one()) {
              const uint32_t to = ring + slot * kStepBytes, bar = full_there + 8 * slot;
              if (rank == 0) mbar_expect_tx(full + 8 * slot, many * 2 * kBoxBytes);
              tma_box(to, &maps.w_in, kb * kBox, n * 64, 2 * pb + rank, bar);
              if (many == 2) tma_box(to + kBoxBytes, &maps.w_in, (kb + 1) * kBox, n * 64, 2 * pb + rank, bar);
            }
            if (++slot == S) slot = 0, phase ^= 1;
          }
        }
    }
    if (abort_flag && rank == 0) {      // copies in flight, the other CTA's too, arrive before the blocks leave
      for (int s = max(step - S, 0); s < step; ++s) mbar_wait_drain(full + 8 * (s % S), (s / S) & 1);
      for (int i = 0; i < p.blocks * (p.pairs == 1 ? 1 : 3); ++i) mbar_wait_drain(kept + 8 * i, (unit & 1) ^ 1);
    }
  } else if (warp == 1 && rank == 0) {
    // products
    int slot = 0;
    uint32_t phase = 0, turn = 0, unit = 0;
    bool ok = true;
    for (int u = blockIdx.x >> 1; u < units && ok; u += stride, ++unit) {
      const int c = u % p.chunks, n_begin = c * p.tiles_n / p.chunks, n_end = (c + 1) * p.tiles_n / p.chunks;
      for (int n = n_begin; n < n_end && ok; ++n, ++turn) {
        const uint32_t buf = turn % kBufs, d = tmem + buf * kBufCols;
        ok = mbar_wait_straight_cluster(acc_empty + 8 * buf, ((turn / kBufs) & 1) ^ 1, &abort_flag);
        tc_fence_after();
        for (int pair = 0; pair < p.pairs; ++pair) {
          const int pa = p.pairs == 1 ? 0 : kPlaneA[pair];
          const bool fetch = n == n_begin && pair < 3, leave = n == n_end - 1 && (p.pairs == 1 || kLastPair[pa] == pair);
          for (int kb = 0; kb < p.blocks && ok; kb += 2) {
            const int many = min(2, p.blocks - kb), at = pa * p.blocks + kb;
            if (fetch)
              for (int j = 0; j < many; ++j) ok = ok && mbar_wait_straight_cluster(kept + 8 * (at + j), unit & 1, &abort_flag);
            ok = ok && mbar_wait_straight_cluster(full + 8 * slot, phase, &abort_flag);
            tc_fence_after();
            const uint32_t a = operand_lo(keep + at * kBlockBytes, 0), b = operand_lo(ring + slot * kStepBytes, 0);
            if (ok && elect_one()) {
              for (int j = 0; j < many; ++j)
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q)
                  mma_pair<true>(d, a + j * (kBlockBytes >> 4) + q * 2, b + j * (kBoxBytes >> 4) + q * 2, p.idesc, (pair | kb | j | (int)q) != 0 ? 1u : 0u);
              mma_commit_pair(empty + 8 * slot);
              if (leave)
                for (int j = 0; j < many; ++j) mma_commit_pair(free_ + 8 * (at + j));
            }
            if (++slot == S) slot = 0, phase ^= 1;
          }
        }
        if (ok && elect_one()) mma_commit_pair(acc_full + 8 * buf);
      }
    }
  } else if (warp >= 4) {
    // accumulators: four warps for each of them, 32 rows and 64 columns to a warp
    const int quad = warp & 3, group = (warp - 4) >> 2, lane = threadIdx.x & 31;
    const uint32_t acc = tmem + group * kBufCols + ((uint32_t)(32 * quad) << 16), empty_there = peer_address(acc_empty + 8 * group, 0);
    constexpr int kWide = sizeof(T) == 2 ? 64 : 32;      // columns of a box
    Outbox box;
    box.open(outs + (warp - 4) * (kHiddenOut / 16), kHiddenOut / 16, 32 * 2 * kWide);
    int turn = 0;
    bool ok = true;
    for (int u = blockIdx.x >> 1; u < units && ok; u += stride) {
      const int m = u / p.chunks, c = u - m * p.chunks, row0 = m * kTileM + rank * (kTileM / 2) + 32 * quad;
      const int n_begin = c * p.tiles_n / p.chunks, n_end = (c + 1) * p.tiles_n / p.chunks;
      for (int nt = n_begin; nt < n_end && ok; ++nt, ++turn) {
        if (turn % kBufs != group) continue;
        ok = mbar_wait_uniform(acc_full + 8 * group, (turn / kBufs) & 1, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        uint32_t at = 0;
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const int n = nt * 64 + q * 16;
          float v[2][16], w[2][16];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            tmem_floats(v[i], acc + (q + i) * 16);
            tmem_floats(w[i], acc + 64 + (q + i) * 16);
          }
          tmem_arrived();
          if (q == 2) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_there(empty_there);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int left = p.cols - n - 16 * i;
            if (p.bias && left > 0) {
              add16<T>(v[i], (const T *)p.bias + n + 16 * i, left, 0);
              add16<T>(w[i], (const T *)p.bias + p.cols + n + 16 * i, left, 0);
            }
            act_values<sizeof(T) == 4, 16>(v[i], p.act);
            multiply<16>(v[i], v[i], w[i]);
          }
          if constexpr (sizeof(T) == 2) {
            if (q == 0) at = box.room();
            box.put<T, 64>(at, q, v[0]);
            box.put<T, 64>(at, q + 1, v[1]);
            if (q == 2) box.send(at, &maps.h, nt * 64, row0, 0);
          } else if (n < p.cols) {
            send_hidden<T>(box, &maps.h, v, n, row0, 0, 1);
          }
        }
      }
    }
    box.close();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (abort_flag) {
    if (warp == 1 && rank == 0) {      // products that are still running end before tensor memory is given back
      if (elect_one()) mma_commit_pair(done);
      __syncwarp();
      mbar_wait_drain(done, 0);
    }
    if (threadIdx.x == 0) report_expired(p.status, p.alarm);
  }
  cluster_sync();                                       // neither leaves while the other may still signal it
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  cluster_sync();
}

// Rows [rows][cols] of float32 as three bfloat16 planes, or 16-bit rows that TMA cannot read as they are (a width or an address
// that is no multiple of 16 bytes), to rows of `pitch` elements: the operands of a call in one launch.
struct PlaneJob {
  const void *src;
  void *dst;
  long long rows;
  int cols, pitch;
  unsigned first;                   // block
};
struct PlaneJobs {
  PlaneJob job[4];
  int many;
};
template <class T>
__global__ void __launch_bounds__(256) ff_planes_kernel(const PlaneJobs jobs) {
  after_previous();
  int j = 0;
  while (j + 1 < jobs.many && blockIdx.x >= jobs.job[j + 1].first) ++j;
  const PlaneJob &s = jobs.job[j];
  const T *src = (const T *)s.src;
  void *dst = s.dst;
  const long long rows = s.rows, t = (long long)(blockIdx.x - s.first) * 256 + threadIdx.x;
  const int cols = s.cols, pitch = s.pitch, per = pitch / 8;
  const long long row = t / per;
  if (row >= rows) return;
  const int c0 = (int)(t - row * per) * 8;
  struct alignas(16) { T v[8]; } k;
  const T *from = src + row * cols + c0;
  if (cols % 8 == 0 && ((uintptr_t)src & 15) == 0) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((int4 *)&k)[i] = ((const int4 *)from)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) k.v[i] = c0 + i < cols ? from[i] : (T)0.f;
  }
  if constexpr (sizeof(T) == 2) {
    *(int4 *)((T *)dst + row * pitch + c0) = *(const int4 *)&k;
  } else {
    const size_t plane = (size_t)rows * pitch;
    __nv_bfloat16 *p = (__nv_bfloat16 *)dst + row * pitch + c0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      uint32_t w[4];
      next_plane<8>(k.v, w, i);
      *(int4 *)(p + i * plane) = *(const int4 *)w;
    }
  }
}

// Sums of shares, in order: out[i] = sum over `parts` of part[k * total + i] (+ bias, residual), for up to five arrays in one launch.
struct SumJob {
  const float *part;
  void *out;
  const void *bias, *residual;      // of rows of `cols` values (or null); out and residual with rows of `pitch`
  int parts, cols, pitch;
  size_t total;                     // values
  unsigned first;                   // block
  int few;                          // few sums of many shares: a warp to each instead of a thread
};
struct SumJobs {
  SumJob job[5];
  int many;
};
template <class T>
__global__ void __launch_bounds__(256) ff_sum_kernel(const SumJobs jobs) {
  after_previous();
  int j = 0;
  while (j + 1 < jobs.many && blockIdx.x >= jobs.job[j + 1].first) ++j;
  const SumJob &s = jobs.job[j];
  float v = 0.f;
  size_t i = (size_t)(blockIdx.x - s.first) * 256 + threadIdx.x;
  if (s.few) {
    i = (size_t)(blockIdx.x - s.first) * 8 + (threadIdx.x >> 5);
    if (i >= s.total) return;
#pragma unroll 4
    for (int k = threadIdx.x & 31; k < s.parts; k += 32) v += s.part[(size_t)k * s.total + i];
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) != 0) return;
  } else {
    if (i >= s.total) return;
#pragma unroll 8
    for (int k = 0; k < s.parts; ++k) v += s.part[(size_t)k * s.total + i];
  }
  size_t at = i;
  if (s.cols != 0) {
    const size_t row = i / (unsigned)s.cols;
    const int col = (int)(i - row * (unsigned)s.cols);
    at = row * s.pitch + col;
    if (s.bias) v += (float)((const T *)s.bias)[col];
    if (s.residual) v += (float)((const T *)s.residual)[at];
  }
  ((T *)s.out)[at] = (T)v;
}

// Column sums of matrices [rows][pitch] (planes of float32 ones added up), a block's share of the rows: part[blockIdx.y * stride + column].
// A thread has eight columns; rows start at multiples of 16 bytes.
struct Columns {
  const void *src;
  int cols, pitch, shares;
  size_t plane, stride;             // planes lie so far apart
  float *part;
};
struct ColumnJobs {
  Columns job[3];
};
template <class T>
__global__ void __launch_bounds__(256) ff_columns_kernel(const ColumnJobs jobs, long long rows, int planes, int accumulate) {
  after_previous();
  __shared__ float sm[256][9];
  const Columns &s = jobs.job[blockIdx.z];
  const int cols = s.cols, pitch = s.pitch;
  if ((int)blockIdx.x * 256 >= cols || (int)blockIdx.y >= s.shares) return;
  const int groups = min((cols + 7) / 8 - (int)blockIdx.x * 32, 32), R = 256 / groups, g = threadIdx.x % groups, w = threadIdx.x / groups, c0 = (blockIdx.x * 32 + g) * 8;
  const long long lo = rows * blockIdx.y / s.shares, hi = rows * (blockIdx.y + 1) / s.shares;
  float v[8] = {};
  if (w < R)
    for (int k = planes - 1; k >= 0; --k) {
      const T *from = (const T *)s.src + k * s.plane + c0;
#pragma unroll 4
      for (long long r = lo + w; r < hi; r += R) {
        struct alignas(16) { T v[8]; } q;
        *(int4 *)&q = *(const int4 *)(from + r * pitch);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += (float)q.v[i];
      }
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) sm[threadIdx.x][i] = v[i];
  __syncthreads();
  for (int t = threadIdx.x; t < groups * 8; t += 256) {
    const int col = blockIdx.x * 256 + t;
    if (col >= cols) continue;
    float sum = 0.f;
    for (int i = 0; i < R; ++i) sum += sm[i * groups + t / 8][t % 8];
    float *o = s.part + blockIdx.y * s.stride + col;
    *o = accumulate ? *o + sum : sum;
  }
}

// Few rows: float32 sums on plain lanes, h never rounded.  A warp takes kFewOutputs outputs of R rows at a time, so that what it loads of the rows serves
// several outputs, and a share of the summed index, so that most loads are under way at once: one latency is what a call of a single row costs.
constexpr int kFewOutputs = 4;
constexpr int kFewRows = 8;        // R at most
constexpr int kFewShares = 8;      // warps to a sum, at most

template <class T, int N>
__device__ __forceinline__ void take(const T *p, int left, int vec, float *v) {
  if (vec) {
    struct alignas(16) { T v[N]; } k;
#pragma unroll
    for (int i = 0; i < N * (int)sizeof(T) / 16; ++i) ((int4 *)&k)[i] = ((const int4 *)p)[i];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)k.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}

// Sums over the lanes of M values: half of them go to the lane across, as long as there are two.
template <int M, int D>
__device__ __forceinline__ void fold(float *v, int lane) {
  if constexpr (M > 1) {
#pragma unroll
    for (int i = 0; i < M / 2; ++i) {
      const float mine = lane & D ? v[i + M / 2] : v[i], other = lane & D ? v[i] : v[i + M / 2];
      v[i] = mine + __shfl_xor_sync(0xffffffffu, other, D);
    }
  } else {
    v[0] += __shfl_xor_sync(0xffffffffu, v[0], D);
  }
  if constexpr (D > 1) fold<(M > 1 ? M / 2 : 1), D / 2>(v, lane);
}

// The sum of w[o][i] x[r][i] over i, for output o and row r (shared memory, every warp of a sum's `shares` has a part): this lane's, of value
// lane % (outputs * R) = o * R + r, in the sum's first warp.  Rows behind `last` are that one.
template <class T, class X, int R>
__device__ __forceinline__ float few_sums(const T *const *w, const X *x, size_t x_stride, int r0, int last, int k, int shares, int vec, float (*parts)[32]) {
  constexpr int N = 16 / sizeof(T), V = kFewOutputs * R;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % shares;
  float acc[V] = {};
  for (int i = (share * 32 + lane) * N; i < k; i += 32 * N * shares) {
    float a[kFewOutputs][N], b[R][N];
#pragma unroll
    for (int o = 0; o < kFewOutputs; ++o) take<T, N>(w[o] + i, k - i, vec, a[o]);
#pragma unroll
    for (int r = 0; r < R; ++r) take<X, N>(x + (size_t)min(r0 + r, last) * x_stride + i, k - i, vec, b[r]);
#pragma unroll
    for (int o = 0; o < kFewOutputs; ++o)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[o * R + r] = fmaf(a[o][e], b[r][e], acc[o * R + r]);
  }
  fold<V, 16>(acc, lane);
  if (lane % (32 / V) == 0) parts[warp][lane / (32 / V)] = acc[0];
  __syncthreads();
  float sum = 0.f;
  if (share == 0)
    for (int q = 0; q < shares; ++q) sum += parts[warp + q][lane % V];
  return sum;
}

template <class T, int R>
__global__ void __launch_bounds__(256) ff_few_hidden_kernel(const T *__restrict__ x, int rows, int c, int hidden, const T *__restrict__ w_in, const T *__restrict__ b_in,
                                                            int act, float *__restrict__ h, int h_stride, int shares, int vec) {
  after_previous();
  __shared__ float parts[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r0 = blockIdx.y * R;
  const int j0 = (blockIdx.x * (blockDim.x / 32 / shares) + warp / shares) * (kFewOutputs / 2);
  const T *w[kFewOutputs];                      // gate and up in turn
#pragma unroll
  for (int o = 0; o < kFewOutputs; ++o) w[o] = w_in + ((size_t)(o & 1) * hidden + min(j0 + o / 2, hidden - 1)) * c;
  const float sum = few_sums<T, T, R>(w, x, c, r0, rows - 1, c, shares, vec, parts), up = __shfl_xor_sync(0xffffffffu, sum, R);
  const int o = lane / R, j = j0 + o / 2, r = r0 + lane % R;
  if (warp % shares != 0 || o >= kFewOutputs || (o & 1) || j >= hidden || r >= rows) return;
  float g = sum + (b_in ? (float)b_in[j] : 0.f);
  act_values<true, 1>(&g, act);
  h[(size_t)r * h_stride + j] = g * (up + (b_in ? (float)b_in[hidden + j] : 0.f));
}

template <class T, int R>
__global__ void __launch_bounds__(256) ff_few_out_kernel(const float *__restrict__ h, int h_stride, int rows, int hidden, int c_out, const T *__restrict__ w_out,
                                                         const T *__restrict__ b_out, const T *__restrict__ residual, T *__restrict__ y, int shares, int vec) {
  after_previous();
  __shared__ float parts[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r0 = blockIdx.y * R;
  const int o0 = (blockIdx.x * (blockDim.x / 32 / shares) + warp / shares) * kFewOutputs;
  const T *w[kFewOutputs];
#pragma unroll
  for (int o = 0; o < kFewOutputs; ++o) w[o] = w_out + (size_t)min(o0 + o, c_out - 1) * hidden;
  float sum = few_sums<T, float, R>(w, h, h_stride, r0, rows - 1, hidden, shares, vec, parts);
  const int o = o0 + lane / R, r = r0 + lane % R;
  if (warp % shares != 0 || lane / R >= kFewOutputs || o >= c_out || r >= rows) return;
  if (b_out) sum += (float)b_out[o];
  const size_t at = (size_t)r * c_out + o;
  if (residual) sum += (float)residual[at];
  y[at] = (T)sum;
}

// ------------------------------------------------------------------------------------------- host
typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult how;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &how) != cudaSuccess || how != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return (EncodeFn)f;
  }();
  return fn;
}

// fn(args...) needs a current context, which a thread has from its first call of the runtime that takes one: a thread of autograd's whose memory comes
// out of a store may get here before.
template <class... A>
CUresult encode(EncodeFn fn, A... args) {
  CUresult r = fn(args...);
  int device;
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = fn(args...);
  return r;
}

// `planes` matrices [rows][cols] with rows of `pitch` elements, one behind the other.
struct Matrix {
  const void *p;
  long long rows;
  int cols, pitch, planes;
};
int make_map(CUtensorMap *map, const Matrix &m, bool f16) {
  const EncodeFn fn = encode_fn();
  if (fn == nullptr) return fail(SSC_ERR_CUDA, "gated_ff: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)m.planes};
  const cuuint64_t strides[2] = {(cuuint64_t)m.pitch * 2, (cuuint64_t)m.pitch * 2 * (cuuint64_t)m.rows};
  const cuuint32_t box[3] = {kBox, kBox, 1}, each[3] = {1, 1, 1};
  const CUresult r = encode(fn, map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(m.p), dims, strides, box, each,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SSC_ERR_CUDA, "gated_ff: no tensor map for [%lld, %d] (error %d)", m.rows, m.cols, (int)r);
  return SSC_OK;
}

// Where boxes of 32 rows and 32 (or 16) columns go; false: rows of this width or at this address cannot be (no error).
bool make_out_map(CUtensorMap *map, const void *p, long long rows, int cols, int pitch, int planes, int type, int width = 32) {
  const int size = type == SSC_PREC_FP32 ? 4 : 2;
  const EncodeFn fn = encode_fn();
  if (fn == nullptr || ((uintptr_t)p & 15) != 0 || pitch * size % 16 != 0) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)pitch * size, (cuuint64_t)pitch * size * (cuuint64_t)rows};
  const cuuint32_t box[3] = {(cuuint32_t)width, 32, 1}, each[3] = {1, 1, 1};
  const CUtensorMapDataType kind = type == SSC_PREC_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == SSC_PREC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(fn, map, kind, 3, const_cast<void *>(p), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, width * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : width * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int pitch_of(int cols) { return (cols + 15) & ~15; }     // rows of whole sectors
int hidden_type(int type) { return type == SSC_PREC_F16 ? SSC_PREC_F16 : SSC_PREC_BF16; }
int planes_for(int type) { return type == SSC_PREC_FP32 ? 3 : 1; }

// Scratch is handed out piece by piece; a null base counts the bytes.
struct Scratch {
  char *base;
  size_t used;
  void *take(size_t bytes) {
    void *p = base ? base + used : nullptr;
    used += align_up(bytes, 256);
    return p;
  }
};

struct Ff {
  int type, n, c, hidden, c_out, act;
  cudaStream_t st;
  int32_t *status;
  int launches;
  PlaneJobs planes;         // operands still to be laid out, and their blocks
  unsigned plane_blocks;
};

// The matrix as TMA reads it: itself, or planes / padded rows in scratch, which lay_out fills.
template <class T>
Matrix operand(Ff &f, Scratch &s, const void *p, long long rows, int cols, int each) {
  const int pitch = pitch_of(cols), planes = planes_for(f.type);
  if (sizeof(T) == 2 && cols % 8 == 0 && ((uintptr_t)p & 15) == 0) return {p, rows / each, cols, cols, each};
  void *to = s.take((size_t)rows * pitch * 2 * planes);
  if (s.base != nullptr) {
    f.planes.job[f.planes.many++] = {p, to, rows, cols, pitch, f.plane_blocks};
    f.plane_blocks += (unsigned)((rows * (pitch / 8) + 255) / 256);
  }
  return {to, rows / each, cols, pitch, planes * each};
}
template <class T>
int lay_out(Ff &f) {
  if (f.planes.many == 0) return SSC_OK;
  const cudaError_t e = launch_ready(ff_planes_kernel<T>, dim3(f.plane_blocks), dim3(256), 0, f.st, f.planes);
  f.planes.many = 0;
  f.plane_blocks = 0;
  ++f.launches;
  return e == cudaSuccess ? SSC_OK : fail(SSC_ERR_CUDA, "gated_ff: %s", cudaGetErrorString(e));
}
// (what operand() may take of the scratch; whether an address is aligned is not known when sizes are asked for)
size_t operand_bytes(int type, long long rows, int cols) { return align_up((size_t)rows * pitch_of(cols) * 2 * planes_for(type), 256); }

uint32_t instruction(const Ff &f, int a_mn, int b_mn, int columns) {
  const uint32_t type = f.type == SSC_PREC_F16 ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(columns >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
}

template <int EPI, class T>
int launch_gemm(Ff &f, const FfMaps &maps, FfParams &p) {
  p.pairs = planes_for(f.type) == 3 ? 6 : 1;
  for (Segment &s : p.seg) s.idesc = instruction(f, s.a_mn, s.b_mn, 2 * s.boxes_b * kBox);
  p.act = f.act;
  p.status = f.status;
  p.alarm = alarm_word();
  const long long tiles = (long long)p.tiles_m * p.tiles_n * p.splits;
  SSC_REQUIRE(tiles < 1ll << 30, "gated_ff: too many tiles");
  const unsigned pairs = (unsigned)(sm_count() / 2), grid = 2 * (tiles < (long long)pairs ? (unsigned)tiles : pairs);
  bool parts = false;
  for (int g = 0; g < p.n_seg; ++g) parts |= p.pairs > 1 && ceil_div(p.seg[g].blocks, p.splits) > kLeave;
  auto kernel = ff_gemm_kernel<EPI, T, false>;
  int threads = kThreads<false>;
  if constexpr (sizeof(T) == 4)
    if (parts) {
      kernel = ff_gemm_kernel<EPI, T, true>;
      threads = kThreads<true>;
    }
  cudaError_t e = allow_smem((const void *)kernel, kSmemBytes<EPI>);
  if (e == cudaSuccess) e = launch_ready(kernel, dim3(grid), dim3(threads), kSmemBytes<EPI>, f.st, maps, p);
  if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "gated_ff: %s", cudaGetErrorString(e));
  ++f.launches;
  return SSC_OK;
}

Segment segment(int k, int boxes_b) {
  Segment s = {};
  s.a_planes = s.b_planes = 1;
  s.blocks = ceil_div(k, kBox);
  s.half_blocks = 1 << 30;
  s.boxes_b = boxes_b;
  return s;
}

// Result tiles of 128 or 256 columns.
int tile_columns(int cols) { return cols <= 128 ? 128 : 256; }

int row_splits(const Ff &f, long long rows, int blocks, int cols);

// C [rows][cols] = A B' (+ bias, residual) as rows of T; B as stored (b_mn: [k][cols]).  part: room for shares of the sum.
template <class T>
int rows_product(Ff &f, const Matrix &a, const Matrix &b, int b_mn, bool halves, int k, int cols, const void *bias, const void *residual, void *out, float *part, int pitch = 0) {
  FfMaps maps = {};
  FfParams p = {};
  if (int e = make_map(&maps.a[0], a, f.type == SSC_PREC_F16)) return e;
  if (int e = make_map(&maps.b[0], b, f.type == SSC_PREC_F16)) return e;
  p.step_n = tile_columns(cols);
  p.seg[0] = segment(k, p.step_n / (2 * kBox));
  p.seg[0].b_mn = b_mn;
  if (halves) {
    p.seg[0].a_half = p.seg[0].b_half = kByK;
    p.seg[0].a_planes = p.seg[0].b_planes = 2;
    p.seg[0].half_blocks = p.seg[0].blocks;
    p.seg[0].blocks *= 2;
  }
  p.n_seg = 1;
  p.rows = (int)a.rows;
  p.cols = cols;
  p.tiles_m = ceil_div(p.rows, kTileM);
  p.m_half = 1 << 30;
  p.tiles_n = ceil_div(cols, p.step_n);
  p.splits = row_splits(f, p.rows, p.seg[0].blocks, cols);
  if (p.splits > 1) {
    const size_t total = (size_t)p.rows * cols;
    p.pitch = cols;
    p.plane = total;
    p.out = part;
    p.boxes = make_out_map(&maps.out[0], part, p.rows, cols, cols, p.splits, SSC_PREC_FP32);
    if (int e = launch_gemm<kPart, T>(f, maps, p)) return e;
    SumJobs jobs = {};
    jobs.many = 1;
    jobs.job[0] = {part, out, bias, residual, p.splits, cols, pitch ? pitch : cols, total, 0, 0};
    const cudaError_t e = launch_ready(ff_sum_kernel<T>, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, f.st, jobs);
    if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "gated_ff: %s", cudaGetErrorString(e));
    ++f.launches;
    return SSC_OK;
  }
  p.pitch = pitch ? pitch : cols;
  p.bias = bias;
  p.residual = residual;
  p.out = out;
  p.vec = p.pitch % (16 / (int)sizeof(T)) == 0 && ((uintptr_t)residual & 15) == 0;
  p.boxes = make_out_map(&maps.out[0], out, p.rows, cols, p.pitch, 1, f.type);
  return launch_gemm<kRows, T>(f, maps, p);
}

// Gate and up with the rows staying in shared memory.
template <class T>
int hidden_product(Ff &f, const Matrix &x, const Matrix &w_in, const void *b_in, void *h) {
  HiddenMaps maps = {};
  HiddenParams p = {};
  const bool f16 = f.type == SSC_PREC_F16;
  if (int e = make_map(&maps.x, x, f16)) return e;
  if (int e = make_map(&maps.w_in, w_in, f16)) return e;
  p.rows = (int)x.rows;
  p.cols = f.hidden;
  if (!make_out_map(&maps.h, h, p.rows, f.hidden, pitch_of(f.hidden), planes_for(f.type), hidden_type(f.type), sizeof(T) == 2 ? 64 : 32))
    return fail(SSC_ERR_CUDA, "gated_ff: no tensor map for the hidden rows");
  p.blocks = ceil_div(f.c, kBox);
  p.pairs = planes_for(f.type) == 3 ? 6 : 1;
  p.tiles_m = ceil_div(p.rows, kTileM);
  p.tiles_n = ceil_div(f.hidden, 64);
  p.act = f.act;
  p.bias = b_in;
  p.idesc = instruction(f, 0, 0, 128);
  p.status = f.status;
  p.alarm = alarm_word();
  const uint32_t fixed = kHiddenOut + (uint32_t)(p.blocks * planes_for(f.type)) * kBlockBytes + 1024;
  p.stages = (int)((kHiddenRoom - fixed) / kStepBytes);
  if (p.stages > kHiddenStages) p.stages = kHiddenStages;
  // as many shares of the columns as make the longest pair's way shortest; rows fetched once more cost about a tile
  const long long pairs = sm_count() / 2;
  long long best = -1;
  for (int c = 1; c <= p.tiles_n && c <= 64; ++c) {
    const long long way = ((long long)p.tiles_m * c + pairs - 1) / pairs * (ceil_div(p.tiles_n, c) + 1);
    if (best < 0 || way < best) best = way, p.chunks = c;
  }
  const long long units = (long long)p.tiles_m * p.chunks;
  const size_t room = fixed + (size_t)p.stages * kStepBytes;
  cudaError_t e = allow_smem((const void *)ff_hidden_kernel<T>, room);
  if (e == cudaSuccess) e = launch_ready(ff_hidden_kernel<T>, dim3((unsigned)(2 * (units < pairs ? units : pairs))), dim3(kHiddenThreads), room, f.st, maps, p);
  if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "gated_ff: %s", cudaGetErrorString(e));
  ++f.launches;
  return SSC_OK;
}

template <class T>
int gate_product(Ff &f, const Matrix &x, const Matrix &w_in, const void *b_in, void *h) {
  if (planes_for(f.type) * ceil_div(f.c, kBox) <= kKeep) return hidden_product<T>(f, x, w_in, b_in, h);
  FfMaps maps = {};
  FfParams p = {};
  if (int e = make_map(&maps.a[0], x, f.type == SSC_PREC_F16)) return e;
  if (int e = make_map(&maps.b[0], w_in, f.type == SSC_PREC_F16)) return e;
  p.step_n = 128;
  p.seg[0] = segment(f.c, p.step_n / kBox);
  p.seg[0].b_half = kByBox;
  p.seg[0].b_planes = 2;
  p.n_seg = 1;
  p.rows = (int)x.rows;
  p.cols = f.hidden;
  p.pitch = pitch_of(f.hidden);
  p.tiles_m = ceil_div(p.rows, kTileM);
  p.m_half = 1 << 30;
  p.tiles_n = ceil_div(f.hidden, p.step_n);
  p.splits = 1;
  p.bias = b_in;
  p.out = h;
  if (!make_out_map(&maps.out[0], h, p.rows, f.hidden, p.pitch, planes_for(f.type), hidden_type(f.type))) return fail(SSC_ERR_CUDA, "gated_ff: no tensor map for the hidden rows");
  return launch_gemm<kGate, T>(f, maps, p);
}

// h, dg and du: gate and up again, and dh = dy Wo.  float32 rows have dh multiplied before: sums that leave tensor memory in between (more than 256 terms)
// are kept in registers, which those of three products exceed.  (Narrower rows could have all three in tensor memory; that form is not there.)
template <class T>
int back_product(Ff &f, const Matrix &x, const Matrix &w_in, const Matrix &gy, const Matrix &w_out, const void *b_in, const float *dh, void *h, void *dgu) {
  FfMaps maps = {};
  FfParams p = {};
  const bool f16 = f.type == SSC_PREC_F16;
  const int g = sizeof(T) == 2 ? 1 : 0;
  if (int e = make_map(&maps.a[g], x, f16)) return e;
  if (int e = make_map(&maps.b[g], w_in, f16)) return e;
  p.step_n = 128;
  p.seg[g] = segment(f.c, 2);
  p.seg[g].b_half = kByBox;
  p.seg[g].b_planes = 2;
  p.n_seg = g + 1;
  if (g == 1) {
    if (int e = make_map(&maps.a[0], gy, f16)) return e;
    if (int e = make_map(&maps.b[0], w_out, f16)) return e;
    p.seg[0] = segment(f.c_out, 1);
    p.seg[0].b_mn = 1;
  }
  p.rows = (int)x.rows;
  p.cols = f.hidden;
  p.pitch = pitch_of(f.hidden);
  p.tiles_m = ceil_div(p.rows, kTileM);
  p.m_half = 1 << 30;
  p.tiles_n = ceil_div(f.hidden, p.step_n);
  p.splits = 1;
  p.bias = b_in;
  p.residual = dh;
  p.out = h;
  p.out2 = dgu;
  const int width = sizeof(T) == 2 ? 32 : 16;      // (float32: nine planes of 16 columns at a time)
  if (!make_out_map(&maps.out[0], h, p.rows, f.hidden, p.pitch, planes_for(f.type), hidden_type(f.type), width) ||
      !make_out_map(&maps.out[1], dgu, p.rows, f.hidden, p.pitch, 2 * planes_for(f.type), hidden_type(f.type), width))
    return fail(SSC_ERR_CUDA, "gated_ff: no tensor map for the hidden rows");
  return launch_gemm<kBack, T>(f, maps, p);
}

// Shares of a long sum: enough tiles for every SM, at least eight blocks of 64 to a share.
int filter_splits(long long rows, int halves, int m, int cols) {
  const int tiles = halves * ceil_div(m, kTileM) * ceil_div(cols, tile_columns(cols)), blocks = ceil_div(rows, kBox);
  int s = sm_count() / 2 / (tiles > 0 ? tiles : 1);
  if (s > blocks / 8) s = blocks / 8;
  return s < 1 ? 1 : s;
}
// part [splits][halves m][cols] (+)= A' B, A [k rows][m] and B [k rows][cols] as stored.
template <class T>
int filter_product(Ff &f, const Matrix &a, const Matrix &b, int halves, int m, int cols, int splits, float *part, int accumulate) {
  FfMaps maps = {};
  FfParams p = {};
  if (int e = make_map(&maps.a[0], a, f.type == SSC_PREC_F16)) return e;
  if (int e = make_map(&maps.b[0], b, f.type == SSC_PREC_F16)) return e;
  p.step_n = tile_columns(cols);
  p.seg[0] = segment((int)a.rows, p.step_n / (2 * kBox));
  p.seg[0].a_mn = p.seg[0].b_mn = 1;
  p.seg[0].a_planes = halves;
  p.seg[0].a_half = halves == 2 ? kByM : kNone;
  p.n_seg = 1;
  p.rows = m;
  p.cols = p.pitch = cols;
  p.plane = (size_t)halves * m * cols;
  p.m_half = ceil_div(m, kTileM);
  p.tiles_m = halves * p.m_half;
  p.tiles_n = ceil_div(cols, p.step_n);
  p.splits = splits;
  p.out = part;
  p.accumulate = accumulate;
  p.boxes = !accumulate && make_out_map(&maps.out[0], part, m, cols, cols, halves * splits, SSC_PREC_FP32);
  return launch_gemm<kPart, T>(f, maps, p);
}

void add_job(SumJobs &jobs, unsigned &blocks, const float *part, int parts, size_t total, void *out, int few) {
  jobs.job[jobs.many++] = {part, out, nullptr, nullptr, parts, 0, 0, total, blocks, few};
  blocks += (unsigned)(few ? (total + 7) / 8 : (total + 255) / 256);
}
// Shares of the rows of a column sum: four blocks to an SM, at least 64 rows to a share.
int column_shares(const Ff &f, long long rows, int cols, int matrices) {
  long long s = 4ll * sm_count() / ((long long)ceil_div(cols, 256) * matrices);
  if (s > rows / 64) s = rows / 64;
  return s < 1 ? 1 : (int)s;
}

// Shares of the sum of a product whose tiles are too few for the pairs of CTAs, or a few too many: what a pair does at the longest, in steps of a
// block (0.3 us), with a dozen for a tile's start and end, and the shares written and read once more (2 MB a step).
int row_splits(const Ff &f, long long rows, int blocks, int cols) {
  const long long pairs = sm_count() / 2, tiles = (long long)ceil_div(rows, kTileM) * ceil_div(cols, tile_columns(cols)), each = planes_for(f.type) == 3 ? 6 : 1;
  long long best = 0;
  int take = 1;
  for (int s = 1; s <= 16 && s <= blocks && (s == 1 || tiles * s <= 4 * pairs); ++s) {
    const long long way = (tiles * s + pairs - 1) / pairs * (ceil_div(blocks, s) * each + 12) + (s > 1 ? 10 + s * rows * cols * 8 / 2000000 : 0);
    if (s == 1 || way < best) best = way, take = s;
  }
  return take;
}
size_t row_split_bytes(const Ff &f, long long rows, int blocks, int cols) {
  const int s = rows > 0 ? row_splits(f, rows, blocks, cols) : 1;
  return s > 1 ? align_up((size_t)s * rows * cols * sizeof(float), 256) : 0;
}

// Rows of one go, so that what lies between the products (planes or rows of h, dg, du, x and dy, dh of float32) is at most a gigabyte: 481 rows
// of the widest there are, a tile or more.
long long rows_at_once(const Ff &f, bool backward) {
  const long long hidden = 2 * planes_for(f.type) * (backward ? 3 : 1) + (backward && f.type == SSC_PREC_FP32 ? 4 : 0);
  const long long per = pitch_of(f.hidden) * hidden + (long long)(pitch_of(f.c) + pitch_of(f.c_out)) * 2 * planes_for(f.type);
  const long long rows = (1ll << 30) / per / kTileM * kTileM;
  return rows < f.n ? rows : f.n;
}

// Room for the shares of the products that give rows (rows_product), for a whole turn of rows and for the last one.
size_t parts_bytes(const Ff &f, long long most, bool back) {
  const long long last = most > 0 ? f.n % most : 0;
  const int c = ceil_div(f.c_out, kBox), h = ceil_div(f.hidden, kBox);
  size_t b = 0;
  for (const long long rows : {most, last}) {
    const size_t one = back ? row_split_bytes(f, rows, 2 * h, f.c) : row_split_bytes(f, rows, h, f.c_out);
    const size_t two = back && f.type == SSC_PREC_FP32 ? row_split_bytes(f, rows, c, f.hidden) : 0;
    if (one > b) b = one;
    if (two > b) b = two;
  }
  return b;
}

// Few rows: products on plain lanes instead of tiles of 256 rows, by what each was measured to take.  Plain lanes: 3.3 us, and for each (up to) eight
// rows the weights at 2.0 (one row), 1.3 (four) or 0.8 (eight) a picosecond in float32, 2.9, 1.5 and 0.7 in 16 bits.  Tiles: 16 us and 10.5 ns
// for each column of x and h in float32, 14 us and 2 ns in 16 bits, whatever the number of rows.  (us, c -> 4 c -> c: float32 8 rows of 256 4.5, 64 rows 13.1, by tiles
// 29.7; 8 rows of 1024 19.7, 64 rows 132, by tiles 85.  bfloat16 1 row of 256 3.7, 16 rows 5.1, by tiles 17; 1 row of 1024 7.5, 16 rows 39, by tiles 24.)
bool few(const Ff &f) {
  if (f.n > kTileM) return false;
  const bool single = f.type == SSC_PREC_FP32;
  const long long weights = (2ll * f.c + f.c_out) * f.hidden, wide = (long long)f.c + f.hidden;
  const long long fs = single ? (f.n == 1 ? 500 : f.n <= 4 ? 790 : 1280) : (f.n == 1 ? 340 : f.n == 2 ? 360 : f.n <= 4 ? 680 : 1400);
  return 3300 + weights * ceil_div(f.n, kFewRows) / 1000 * fs / 1000 < (single ? 16000 + 21 * wide / 2 : 14000 + 2 * wide);
}

// Warps that share a sum of k terms: a piece to a lane each where that takes no more than kFewShares of them.
int few_shares(int k, int piece) {
  int s = 1;
  while (s < kFewShares && s * 32 * piece < k) s *= 2;
  return s;
}
template <class T, int R>
cudaError_t few_rows(const Ff &f, const void *x, const void *w_in, const void *w_out, const void *b_in, const void *b_out, const void *residual, float *h, int h_stride,
                     void *out) {
  constexpr int N = 16 / (int)sizeof(T);
  const int vec_in = f.c % N == 0 && (((uintptr_t)w_in | (uintptr_t)x) & 15) == 0, vec_out = f.hidden % N == 0 && ((uintptr_t)w_out & 15) == 0;
  const int shares_in = few_shares(f.c, N), shares_out = few_shares(f.hidden, N), warps_in = shares_in < 4 ? 4 : shares_in, warps_out = shares_out < 4 ? 4 : shares_out;
  const int rows = ceil_div(f.n, R);
  cudaError_t e = launch_ready(ff_few_hidden_kernel<T, R>, dim3(ceil_div(f.hidden, kFewOutputs / 2 * (warps_in / shares_in)), rows), dim3(32 * warps_in), 0, f.st, (const T *)x, f.n,
                               f.c, f.hidden, (const T *)w_in, (const T *)b_in, f.act, h, h_stride, shares_in, vec_in);
  if (e == cudaSuccess)
    e = launch_ready(ff_few_out_kernel<T, R>, dim3(ceil_div(f.c_out, kFewOutputs * (warps_out / shares_out)), rows), dim3(32 * warps_out), 0, f.st, (const float *)h, h_stride, f.n,
                     f.hidden, f.c_out, (const T *)w_out, (const T *)b_out, (const T *)residual, (T *)out, shares_out, vec_out);
  return e;
}

template <class T>
int forward(Ff &f, Scratch s, const void *x, const void *w_in, const void *w_out, const void *b_in, const void *b_out, const void *residual, void *out) {
  if (few(f)) {
    const int h_stride = (f.hidden + 3) & ~3;
    float *h = (float *)s.take((size_t)f.n * h_stride * sizeof(float));
    const cudaError_t e = f.n == 1   ? few_rows<T, 1>(f, x, w_in, w_out, b_in, b_out, residual, h, h_stride, out)
                          : f.n == 2 ? few_rows<T, 2>(f, x, w_in, w_out, b_in, b_out, residual, h, h_stride, out)
                          : f.n <= 4 ? few_rows<T, 4>(f, x, w_in, w_out, b_in, b_out, residual, h, h_stride, out)
                                     : few_rows<T, kFewRows>(f, x, w_in, w_out, b_in, b_out, residual, h, h_stride, out);
    if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "gated_ff_fwd: %s", cudaGetErrorString(e));
    f.launches += 2;
    return SSC_OK;
  }
  const Matrix wi = operand<T>(f, s, w_in, 2ll * f.hidden, f.c, 2), wo = operand<T>(f, s, w_out, f.c_out, f.hidden, 1);
  const long long most = rows_at_once(f, false);
  const int pitch = pitch_of(f.hidden), planes = planes_for(f.type);
  void *h = s.take((size_t)most * pitch * 2 * planes);
  float *part = (float *)s.take(parts_bytes(f, most, false));
  for (long long r = 0; r < f.n; r += most) {
    const long long rows = f.n - r < most ? f.n - r : most;
    Scratch here = s;
    const Matrix xm = operand<T>(f, here, (const T *)x + r * f.c, rows, f.c, 1);
    if (int e = lay_out<T>(f)) return e;
    if (int e = gate_product<T>(f, xm, wi, b_in, h)) return e;
    const Matrix hm = {h, rows, f.hidden, pitch, planes};
    if (int e = rows_product<T>(f, hm, wo, 0, false, f.hidden, f.c_out, b_out, residual ? (const T *)residual + r * f.c_out : nullptr, (T *)out + r * f.c_out, part)) return e;
  }
  return SSC_OK;
}

template <class T>
int backward(Ff &f, Scratch s, const void *x, const void *gy, const void *w_in, const void *w_out, const void *b_in, void *gx, void *gw_in, void *gw_out, void *gb_in,
             void *gb_out) {
  const Matrix wi = operand<T>(f, s, w_in, 2ll * f.hidden, f.c, 2), wo = operand<T>(f, s, w_out, f.c_out, f.hidden, 1);
  using U = std::conditional_t<sizeof(T) == 4, __nv_bfloat16, T>;
  const long long most = rows_at_once(f, true);
  const int pitch = pitch_of(f.hidden), planes = planes_for(f.type);
  const size_t size_in = 2 * (size_t)f.hidden * f.c, size_out = (size_t)f.c_out * f.hidden;
  const int split_in = filter_splits(most, 2, f.hidden, f.c), split_out = filter_splits(most, 1, f.c_out, f.hidden);
  void *h = s.take((size_t)most * pitch * 2 * planes), *dgu = s.take((size_t)most * pitch * 4 * planes);
  float *dh = planes == 3 ? (float *)s.take((size_t)most * pitch * sizeof(float)) : nullptr;
  float *part_in = (float *)s.take(split_in * size_in * sizeof(float)), *part_out = (float *)s.take(split_out * size_out * sizeof(float));
  const int shares_in = column_shares(f, most, f.hidden, 2), shares_out = column_shares(f, most, f.c_out, 1);
  float *cols_in = (float *)s.take((size_t)shares_in * 2 * f.hidden * sizeof(float)), *cols_out = (float *)s.take((size_t)shares_out * f.c_out * sizeof(float));
  float *part = (float *)s.take(parts_bytes(f, most, true));
  for (long long r = 0; r < f.n; r += most) {
    const long long rows = f.n - r < most ? f.n - r : most;
    Scratch here = s;
    const int more = r > 0;
    const Matrix xm = operand<T>(f, here, (const T *)x + r * f.c, rows, f.c, 1), gm = operand<T>(f, here, (const T *)gy + r * f.c_out, rows, f.c_out, 1);
    if (int k = lay_out<T>(f)) return k;
    if (dh)
      if (int k = rows_product<T>(f, gm, wo, 1, false, f.c_out, f.hidden, nullptr, nullptr, dh, part, pitch)) return k;
    if (int k = back_product<T>(f, xm, wi, gm, wo, b_in, dh, h, dgu)) return k;
    const Matrix hm = {h, rows, f.hidden, pitch, planes}, dm = {dgu, rows, f.hidden, pitch, 2 * planes};
    if (gx)
      if (int k = rows_product<T>(f, dm, wi, 1, true, f.hidden, f.c, nullptr, nullptr, (T *)gx + r * f.c, part)) return k;
    if (gw_in)
      if (int k = filter_product<T>(f, dm, xm, 2, f.hidden, f.c, split_in, part_in, more)) return k;
    if (gw_out)
      if (int k = filter_product<T>(f, gm, hm, 1, f.c_out, f.hidden, split_out, part_out, more)) return k;
    const size_t plane = (size_t)rows * pitch;
    if (gb_in || gb_out) {
      ColumnJobs jobs = {};
      int many = 0;
      for (int i = 0; gb_in && i < 2; ++i)
        jobs.job[many++] = {(const U *)dgu + i * plane, f.hidden, pitch, shares_in, planes == 3 ? 2 * plane : 0, 2 * (size_t)f.hidden, cols_in + (size_t)i * f.hidden};
      if (gb_out) jobs.job[many++] = {gm.p, f.c_out, gm.pitch, shares_out, (size_t)rows * gm.pitch, (size_t)f.c_out, cols_out};
      const int widest = gb_in && (!gb_out || f.hidden > f.c_out) ? f.hidden : f.c_out;
      const int shares = gb_in && (!gb_out || shares_in > shares_out) ? shares_in : shares_out;
      const cudaError_t e = launch_ready(ff_columns_kernel<U>, dim3(ceil_div(widest, 256), shares, many), dim3(256), 0, f.st, jobs, rows, planes, more);
      if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "gated_ff_bwd: %s", cudaGetErrorString(e));
      ++f.launches;
    }
  }
  SumJobs jobs = {};
  unsigned blocks = 0;
  if (gw_in) add_job(jobs, blocks, part_in, split_in, size_in, gw_in, 0);
  if (gw_out) add_job(jobs, blocks, part_out, split_out, size_out, gw_out, 0);
  if (gb_in) add_job(jobs, blocks, cols_in, shares_in, 2 * (size_t)f.hidden, gb_in, 1);
  if (gb_out) add_job(jobs, blocks, cols_out, shares_out, f.c_out, gb_out, 1);
  if (blocks > 0) {
    const cudaError_t e = launch_ready(ff_sum_kernel<T>, dim3(blocks), dim3(256), 0, f.st, jobs);
    if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "gated_ff_bwd: %s", cudaGetErrorString(e));
    ++f.launches;
  }
  return SSC_OK;
}

size_t scratch_bytes_for(const Ff &f, bool back) {
  if (!back && few(f)) return align_up((size_t)f.n * ((f.hidden + 3) & ~3) * sizeof(float), 256) + 256;
  const long long most = rows_at_once(f, back);
  const size_t hidden = align_up((size_t)most * pitch_of(f.hidden) * 2 * planes_for(f.type), 256);
  size_t b = 256 + operand_bytes(f.type, 2ll * f.hidden, f.c) + operand_bytes(f.type, f.c_out, f.hidden) + operand_bytes(f.type, most, f.c);
  if (!back) return b + hidden + parts_bytes(f, most, false);
  const size_t size_in = 2 * (size_t)f.hidden * f.c, size_out = (size_t)f.c_out * f.hidden;
  b += operand_bytes(f.type, most, f.c_out) + 3 * hidden + 512 + (f.type == SSC_PREC_FP32 ? align_up((size_t)most * pitch_of(f.hidden) * sizeof(float), 256) : 0);
  b += align_up(filter_splits(most, 2, f.hidden, f.c) * size_in * 4, 256) + align_up(filter_splits(most, 1, f.c_out, f.hidden) * size_out * 4, 256);
  b += parts_bytes(f, most, true);
  return b + align_up((size_t)column_shares(f, most, f.hidden, 2) * 8 * f.hidden, 256) + align_up((size_t)column_shares(f, most, f.c_out, 1) * 4 * f.c_out, 256);
}

constexpr int kMostChannels = 65536;
int ff_check(const Ff &f, const char *what) {
  SSC_REQUIRE(f.type == SSC_PREC_FP32 || f.type == SSC_PREC_F16 || f.type == SSC_PREC_BF16, "%s: unknown type", what);
  SSC_REQUIRE(f.n >= 0 && f.n <= 1 << 30 && f.c >= 1 && f.hidden >= 1 && f.c_out >= 1 && f.c <= kMostChannels && f.hidden <= kMostChannels && f.c_out <= kMostChannels, "%s: bad sizes", what);
  SSC_REQUIRE(f.act >= 0 && f.act <= 4, "%s: unknown activation", what);
  return SSC_OK;
}

}  // namespace
}  // namespace ssc

extern "C" size_t ssc_gated_ff_scratch_bytes(int type, int n, int c, int hidden, int c_out, int backward) {
  ssc::Ff f = {type, n, c, hidden, c_out, 0};
  if (ssc::ff_check(f, "gated_ff_scratch_bytes") != SSC_OK) return 0;
  return ssc::scratch_bytes_for(f, backward != 0);
}

extern "C" int ssc_gated_ff_fwd(const void *x, int type, int n, int c, int hidden, int c_out, const void *w_in, const void *w_out, const void *b_in, const void *b_out,
                                const void *residual, int act, void *out, int32_t *status, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace ssc;
  Ff f = {type, n, c, hidden, c_out, act, as_stream(stream), status, 0, {}, 0};
  if (int e = ff_check(f, "gated_ff_fwd")) return e;
  SSC_REQUIRE(w_in && w_out && (n == 0 || (x && out)), "gated_ff_fwd: null pointer");
  if (n == 0) return SSC_OK;
  if (scratch == nullptr || ((uintptr_t)scratch & 15) != 0 || scratch_bytes < scratch_bytes_for(f, false)) return fail(SSC_ERR_SCRATCH, "gated_ff_fwd: scratch too small");
  const Scratch s = {(char *)(((uintptr_t)scratch + 255) & ~(uintptr_t)255), 0};
  int e = type == SSC_PREC_FP32  ? forward<float>(f, s, x, w_in, w_out, b_in, b_out, residual, out)
          : type == SSC_PREC_F16 ? forward<__half>(f, s, x, w_in, w_out, b_in, b_out, residual, out)
                                 : forward<__nv_bfloat16>(f, s, x, w_in, w_out, b_in, b_out, residual, out);
  note_launches(f.launches);
  if (e != SSC_OK) return e;
  SSC_CHECK_LAUNCH("gated_ff_fwd");
  return SSC_OK;
}

extern "C" int ssc_gated_ff_bwd(const void *x, const void *gy, int type, int n, int c, int hidden, int c_out, const void *w_in, const void *w_out, const void *b_in, int act,
                                void *gx, void *gw_in, void *gw_out, void *gb_in, void *gb_out, int32_t *status, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace ssc;
  Ff f = {type, n, c, hidden, c_out, act, as_stream(stream), status, 0, {}, 0};
  if (int e = ff_check(f, "gated_ff_bwd")) return e;
  SSC_REQUIRE(w_in && w_out && (n == 0 || (x && gy)), "gated_ff_bwd: null pointer");
  if (n == 0) {
    const size_t size = type == SSC_PREC_FP32 ? 4 : 2;
    cudaError_t e = cudaSuccess;
    if (gw_in) e = cudaMemsetAsync(gw_in, 0, 2 * (size_t)hidden * c * size, f.st);
    if (gw_out && e == cudaSuccess) e = cudaMemsetAsync(gw_out, 0, (size_t)c_out * hidden * size, f.st);
    if (gb_in && e == cudaSuccess) e = cudaMemsetAsync(gb_in, 0, 2 * (size_t)hidden * size, f.st);
    if (gb_out && e == cudaSuccess) e = cudaMemsetAsync(gb_out, 0, (size_t)c_out * size, f.st);
    if (e != cudaSuccess) return fail(SSC_ERR_CUDA, "gated_ff_bwd: %s", cudaGetErrorString(e));
    return SSC_OK;
  }
  if (scratch == nullptr || ((uintptr_t)scratch & 15) != 0 || scratch_bytes < scratch_bytes_for(f, true)) return fail(SSC_ERR_SCRATCH, "gated_ff_bwd: scratch too small");
  const Scratch s = {(char *)(((uintptr_t)scratch + 255) & ~(uintptr_t)255), 0};
  int e = type == SSC_PREC_FP32  ? backward<float>(f, s, x, gy, w_in, w_out, b_in, gx, gw_in, gw_out, gb_in, gb_out)
          : type == SSC_PREC_F16 ? backward<__half>(f, s, x, gy, w_in, w_out, b_in, gx, gw_in, gw_out, gb_in, gb_out)
                                 : backward<__nv_bfloat16>(f, s, x, gy, w_in, w_out, b_in, gx, gw_in, gw_out, gb_in, gb_out);
  note_launches(f.launches);
  if (e != SSC_OK) return e;
  SSC_CHECK_LAUNCH("gated_ff_bwd");
  return SSC_OK;
}
