// linear_tc.cu -- the linear layer's products on the tensor cores.
//
//   D[row][chan] = sum_k A(chan, k) B(row, k)
//
// Output channels (the contiguous index of the output) lie on the MMA's M side, so that they are
// TMEM lanes: a warp stores 32 consecutive channels of one row at a time, whatever the row stride
// and alignment, and needs no staging tile.  The product's rows are the MMA's N side, in tiles of
// 16 to 256 columns, so that a few tokens do not pay for a full tile.
//
// Each operand is read by TMA either along k (its rows are the product's index, "K-major") or
// across it (its rows are k, "MN-major"): the tensor core takes both, so the gradients' transposed
// operands need no transposed copies.
//
//   forward   A = W   [out][in] K-major    B = x    [rows][in]  K-major
//   dx        A = W   [out][in] MN-major   B = dpre [rows][out] K-major
//   dW        A = x   [rows][in] MN-major  B = dpre [rows][out] MN-major
//
// bf16 and fp16 run as they are (one plane).  An fp32 operand is the sum of three bf16 planes
// (3 x 8 significant bits; the differences are exact), and the product is the six plane products
// that reach 2^-24 of it: a3 b1, a1 b3, a2 b2, a2 b1, a1 b2, a1 b1, smallest first.  The tensor
// core's fp32 accumulator truncates each addition, which would bias a long sum, so every chunk of
// k starts a new accumulator and the epilogue warps add the chunks in registers, rounding to
// nearest.
//
// One CTA per SM walks its tiles: a TMA producer warp, an MMA warp, eight epilogue warps.  Two
// accumulators in TMEM let the epilogue of one tile run beside the next tile's MMAs.  When there
// are fewer tiles than SMs, a cluster of CTAs shares a tile's k range: each leaves its part in its
// shared memory and adds a slice of the columns from all of them through distributed shared
// memory, in the order of the parts.
#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "linear_tc.cuh"
#include "ptx.cuh"

using namespace ptb;

namespace ptb {
int tensor_map_encoder(PFN_cuTensorMapEncodeTiled_v12000 *fn);   // conv_tc.cu
}

namespace {

constexpr int kEpiWarps = 8;
constexpr int kTcThreads = (4 + kEpiWarps) * 32;   // warp 0 TMA, warp 1 MMA, 2-3 idle, 4-11 epilogue
constexpr int kM = 128;
constexpr int kMaxStages = 10;
constexpr int kSmemBudget = 217 * 1024;
constexpr int kSmemBytes = kSmemBudget + 1024 + 512;

struct TcArgs {
  LinearEpi e;
  int64_t rows, chans;      // output rows (N side) and channels (M side)
  int kiters;               // k stages in all
  int split;                // CTAs that share a tile's k range (the cluster)
  int per;                  // k stages of one of them
  int bn;                   // rows per tile
  int stages;
  int tiles_m, tiles_n;     // channel tiles, row tiles
  uint32_t idesc;
  bool a_mn, b_mn;
};

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Shared-memory descriptors.  K-major: rows of KB elements (128 or 64 bytes, swizzled by as much),
// 8-row atoms one after another.  MN-major: blocks of 64 elements (128 bytes, swizzled) x KB k
// rows; `lead` bytes from one block of 64 to the next, 8 k rows to an atom of 1024 bytes.
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lead, uint32_t atom, uint32_t swizzle) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>((atom >> 4) & 0x3FFFu) << 32 | static_cast<uint64_t>(1u) << 46 |
         static_cast<uint64_t>(swizzle) << 61;
}

// Tile t of the walk: channel tiles fastest inside bands of 16, so that concurrent CTAs share both
// operands through L2.
__device__ __forceinline__ void tile_at(const TcArgs &g, int t, int *tm, int *tn) {
  constexpr int kBand = 16;
  const int band = t / (kBand * g.tiles_n);
  const int left = g.tiles_m - band * kBand;
  const int height = left < kBand ? left : kBand;
  const int in = t - band * kBand * g.tiles_n;
  *tm = band * kBand + in % height;
  *tn = in / height;
}

// Sixteen results of one channel, rows row0 .. row0 + 15: bias, activation, residual, store.
template <class T>
__device__ __forceinline__ void emit16(const TcArgs &g, float (&v)[16], int64_t chan, int64_t row0, float bias) {
  const LinearEpi &e = g.e;
  const int n = static_cast<int>(min(static_cast<int64_t>(16), g.rows - row0));
  if (chan >= g.chans || n <= 0) return;
  float r[16];
  if (e.residual) {
    const T *p = static_cast<const T *>(e.residual) + row0 * e.ldr + chan;
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = j < n ? to_f32(p[j * e.ldr]) : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] += bias;
  if (e.pre) {
    T *p = static_cast<T *>(e.pre) + row0 * e.ldp + chan;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < n) p[j * e.ldp] = from_f32<T>(v[j]);
  }
  if (e.act) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = act_value(v[j], e.act, e.slope);
  }
  if (e.residual) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += r[j];
  }
  T *p = static_cast<T *>(e.y) + row0 * e.ldy + chan;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < n) p[j * e.ldy] = from_f32<T>(v[j]);
}

// P planes per operand, KB elements of k per stage.
template <class T, int P, int KB>
__global__ void __launch_bounds__(kTcThreads, 1)
    linear_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const TcArgs g, uint32_t *gerr) {
  namespace cg = cooperative_groups;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *gbase = smem_raw + (base - raw);
  const uint32_t a_plane = kM * KB * 2, b_plane = static_cast<uint32_t>(g.bn) * KB * 2;
  const uint32_t stage_bytes = P * (a_plane + b_plane);
  const uint32_t bar0 = base + kSmemBudget;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kMaxStages + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kMaxStages + 2 + b); };
  const uint32_t drain = bar0 + 8u * (2 * kMaxStages + 4);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(gbase + kSmemBudget + 8 * (2 * kMaxStages + 5));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // accumulators are a power of two of columns apart, TMEM is allocated in powers of two from 32
  uint32_t acc_cols = 16;
  while (acc_cols < static_cast<uint32_t>(g.bn)) acc_cols *= 2;
  const uint32_t tmem_cols = 2 * acc_cols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int rank = static_cast<int>(blockIdx.x) % g.split;
  const int step = static_cast<int>(gridDim.x) / g.split;
  const int tiles = g.tiles_m * g.tiles_n;
  const int k_lo = rank * g.per, k_hi = min(k_lo + g.per, g.kiters);
  // stages per accumulator: all of them, or (three planes) a chunk of 64 elements of k
  const int chunk = P == 1 ? g.per : 64 / KB;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer
    int s = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x / g.split; t < tiles && ok; t += step) {
      int tm, tn;
      tile_at(g, t, &tm, &tn);
      for (int k = k_lo; k < k_hi; ++k) {
        if (issued >= g.stages && !mbar_wait(empty(s), phase ^ 1u, abort_flag, gerr, ERR_WAIT_EMPTY)) {
          ok = false;
          break;
        }
        const uint32_t a0 = base + s * stage_bytes, b0 = a0 + P * a_plane;
        mbar_expect_tx(full(s), stage_bytes);
        for (int p = 0; p < P; ++p) {
          if (g.a_mn) {
            for (int i = 0; i < kM / 64; ++i)
              tma_load_3d(a0 + p * a_plane + i * KB * 128, &map_a, full(s), tm * kM + i * 64, k * KB, p);
          } else {
            tma_load_3d(a0 + p * a_plane, &map_a, full(s), k * KB, tm * kM, p);
          }
          if (g.b_mn) {
            for (int i = 0; i < g.bn / 64; ++i)
              tma_load_3d(b0 + p * b_plane + i * KB * 128, &map_b, full(s), tn * g.bn + i * 64, k * KB, p);
          } else {
            tma_load_3d(b0 + p * b_plane, &map_b, full(s), k * KB, tn * g.bn, p);
          }
        }
        ++issued;
        if (++s == g.stages) s = 0, phase ^= 1u;
      }
    }
    if (!ok) {   // copies in flight must land before the CTA's shared memory is given up
      const int flying = min(issued, g.stages);
      for (int i = 0; i < flying; ++i) {
        if (s == 0) s = g.stages, phase ^= 1u;
        --s;
        uint32_t it = 0;
        while (!mbar_try_wait(full(s), phase) && ++it < kWaitLimit) {
        }
        if (it >= kWaitLimit) atomicOr(gerr, ERR_WAIT_DRAIN);
      }
    }
  } else if (warp == 1 && lane == 0) {
    // ---------------- MMA issuer
    constexpr uint32_t kSwz = KB == 64 ? 2u : 4u;              // 128- or 64-byte swizzle, K-major
    constexpr uint32_t kAtom = KB * 16;                        // 8 rows of KB elements
    const uint32_t a_adv = g.a_mn ? 2048u >> 4 : 32u >> 4;     // 16 elements of k further on
    const uint32_t b_adv = g.b_mn ? 2048u >> 4 : 32u >> 4;
    int s = 0, unit = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x / g.split; t < tiles && ok; t += step) {
      for (int k = k_lo; k < k_hi && ok; ++unit) {
        const int b = unit & 1;
        if (unit >= 2 && !mbar_wait(acc_empty(b), ((unit >> 1) & 1) ^ 1u, abort_flag, gerr, ERR_WAIT_ACC)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + b * acc_cols;
        const int k_end = min(k + chunk, k_hi);
        uint32_t accumulate = 0;
        for (; k < k_end; ++k) {
          if (!mbar_wait(full(s), phase, abort_flag, gerr, ERR_WAIT_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = base + s * stage_bytes, b0 = a0 + P * a_plane;
#pragma unroll
          for (int q = 0; q < (P == 1 ? 1 : 6); ++q) {
            constexpr int kPa[6] = {2, 0, 1, 1, 0, 0}, kPb[6] = {0, 2, 1, 0, 1, 0};
            const uint32_t ap = a0 + (P == 1 ? 0 : kPa[q]) * a_plane, bp = b0 + (P == 1 ? 0 : kPb[q]) * b_plane;
            const uint64_t da = g.a_mn ? sdesc(ap, KB * 128, 1024, 2) : sdesc(ap, 16, kAtom, kSwz);
            const uint64_t db = g.b_mn ? sdesc(bp, KB * 128, 1024, 2) : sdesc(bp, 16, kAtom, kSwz);
#pragma unroll
            for (int i = 0; i < KB / 16; ++i) {
              mma_f16(d, da + i * a_adv, db + i * b_adv, g.idesc, accumulate);
              accumulate = 1;
            }
          }
          mma_commit(empty(s));
          if (++s == g.stages) s = 0, phase ^= 1u;
        }
        if (ok) mma_commit(acc_full(b));
      }
    }
    if (!ok) {   // MMAs already issued must finish before TMEM is released
      mma_commit(drain);
      uint32_t it = 0;
      while (!mbar_try_wait(drain, 0) && ++it < kWaitLimit) {
      }
      if (it >= kWaitLimit) atomicOr(gerr, ERR_WAIT_DRAIN);
    }
  } else if (warp >= 4) {
    // ---------------- epilogue warps: lanes 32 (warp % 4) .. + 31, every other block of 16 columns
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t tl = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    int unit = 0;
    bool ok = true;
    for (int t = blockIdx.x / g.split; t < tiles && ok; t += step) {
      int tm, tn;
      tile_at(g, t, &tm, &tn);
      const int64_t chan = static_cast<int64_t>(tm) * kM + quad * 32 + lane;
      const int64_t row0 = static_cast<int64_t>(tn) * g.bn;
      const float bias = g.e.bias && chan < g.chans ? to_f32(static_cast<const T *>(g.e.bias)[chan]) : 0.0f;
      float *part = reinterpret_cast<float *>(gbase);   // split: [bn][128] of this CTA's part
      if constexpr (P == 1) {
        const int b = unit & 1;
        if (!mbar_wait(acc_full(b), (unit >> 1) & 1, abort_flag, gerr, ERR_WAIT_ACC)) break;
        tc_fence_after();
        for (int c = half * 16; c < g.bn; c += 32) {
          float v[16];
          tmem_ld16(tl + b * acc_cols + c, v);
          if (g.split > 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(c + j) * kM + quad * 32 + lane] = v[j];
          } else {
            emit16<T>(g, v, chan, row0 + c, bias);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty(b));
        ++unit;
      } else {
        float acc[8][16];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
        for (int k = k_lo; k < k_hi && ok; k += chunk, ++unit) {
          const int b = unit & 1;
          if (!mbar_wait(acc_full(b), (unit >> 1) & 1, abort_flag, gerr, ERR_WAIT_ACC)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (half * 16 + i * 32 < g.bn) {
              float v[16];
              tmem_ld16(tl + b * acc_cols + half * 16 + i * 32, v);
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[i][j] += v[j];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty(b));
        }
        if (!ok) break;
        if (g.split > 1) {
          // the stages still hold operands of the last chunk until its MMAs are done, which the
          // last accumulator's arrival says
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (half * 16 + i * 32 < g.bn)
#pragma unroll
              for (int j = 0; j < 16; ++j)
                part[(half * 16 + i * 32 + j) * kM + quad * 32 + lane] = acc[i][j];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (half * 16 + i * 32 < g.bn) emit16<T>(g, acc[i], chan, row0 + half * 16 + i * 32, bias);
        }
      }
    }
  }
  if (g.split > 1) {
    // ---------------- one tile per cluster: add the parts, a slice of the rows per CTA
    __syncwarp();
    auto cluster = cg::this_cluster();
    cluster.sync();
    const int t = blockIdx.x / g.split;
    if (warp >= 4 && !*abort_flag) {
      const int quad = warp & 3, half = (warp - 4) >> 2;
      int tm, tn;
      tile_at(g, t, &tm, &tn);
      const int64_t chan = static_cast<int64_t>(tm) * kM + quad * 32 + lane;
      float *part = reinterpret_cast<float *>(gbase);
      const int width = g.bn / g.split;
      for (int c = rank * width + half; c < (rank + 1) * width; c += 2) {
        const int64_t row = static_cast<int64_t>(tn) * g.bn + c;
        float v = 0.0f;
        for (int r = 0; r < g.split; ++r) v += cluster.map_shared_rank(part, r)[c * kM + quad * 32 + lane];
        if (chan < g.chans && row < g.rows) linear_store<T>(g.e, row, chan, v);
      }
    }
    cluster.sync();   // no CTA leaves while another still reads its part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------------------------------------------ operand planes
// A matrix copied into the rows and planes the tensor cores read.
template <class T>
__global__ void __launch_bounds__(256) pack_kernel(const PackArgs a) {
  const int64_t cols8 = a.ld_out;
  const int64_t total = a.rows * cols8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / cols8, c = i % cols8;
    if (c >= a.cols) continue;
    const T v = static_cast<const T *>(a.src)[r * a.ld + c];
    if constexpr (sizeof(T) == 4) {
      __nv_bfloat16 o[3];
      split3(v, o);
#pragma unroll
      for (int p = 0; p < 3; ++p) static_cast<__nv_bfloat16 *>(a.dst)[p * a.plane + i] = o[p];
    } else {
      static_cast<T *>(a.dst)[i] = v;
    }
  }
}

int encode(CUtensorMap *m, const TcOperand &o, bool half, int planes, int box_inner, int box_outer, bool swz64) {
  PFN_cuTensorMapEncodeTiled_v12000 enc;
  if (tensor_map_encoder(&enc)) return -1;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(planes > 1 ? o.plane * 2 : 16)};
  cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                         const_cast<void *>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swz64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  PTB_REQUIRE(r == CUDA_SUCCESS, "pt_b200: operand tensor map encode failed (%d)", (int)r);
  return 0;
}

// Tile height and k split: the cheapest of the candidates by a count of SM clocks.  A stage of 64
// elements of k takes the longer of its MMAs (bn / 2 clocks for 16 of k) and of its bytes at the
// L2's share of one SM; a tile adds its start, its epilogue and, when its k range is shared, the
// exchange of the parts.
struct Shape {
  int bn, split;
};
Shape pick_shape(int sms, int64_t rows, int64_t chans, int kiters, int kb, int planes, bool b_mn) {
  Shape best{0, 1};
  double best_cost = 0;
  const int64_t tm = (chans + kM - 1) / kM;
  const int products = planes == 1 ? 1 : 6;
  for (int bn : {16, 32, 64, 128, 256}) {
    if (b_mn && bn < 64) continue;
    const int64_t tiles = tm * ((rows + bn - 1) / bn);
    for (int split : {1, 2, 4, 8}) {
      const int per = (kiters + split - 1) / split;
      if (split > 1 && ((split - 1) * per >= kiters || tiles * split > sms)) continue;
      const double mma = products * (kb / 16) * std::max(bn / 2.0, 16.0);
      const double load = planes * kb * 2.0 * (kM + bn) / 60.0;
      const double tail = 600.0 + bn * (split > 1 ? 8.0 + 6.0 * split : 8.0);
      const int64_t waves = (tiles * split + sms - 1) / sms;
      const double cost = 2000.0 + waves * (per * std::max(mma, load)) + tail;
      if (!best.bn || cost < best_cost) best = Shape{bn, split}, best_cost = cost;
    }
  }
  return best;
}

template <class T, int P, int KB>
int launch(const pt_b200_ops *h, const TcProduct &p, cudaStream_t st) {
  TcArgs g{};
  g.e = p.e;
  g.rows = p.rows;
  g.chans = p.chans;
  g.a_mn = p.a_mn;
  g.b_mn = p.b_mn;
  g.kiters = static_cast<int>((p.k + KB - 1) / KB);
  const Shape sh = pick_shape(h->sms, p.rows, p.chans, g.kiters, KB, P, p.b_mn);
  g.bn = sh.bn;
  g.split = sh.split;
  g.per = (g.kiters + g.split - 1) / g.split;
  const int stage = P * (kM + g.bn) * KB * 2;
  g.stages = std::min(kMaxStages, kSmemBudget / stage);
  g.tiles_m = static_cast<int>((p.chans + kM - 1) / kM);
  const int64_t tiles_n = (p.rows + g.bn - 1) / g.bn;
  PTB_REQUIRE(tiles_n * g.tiles_m < (int64_t(1) << 30), "pt_b200: product of %lld x %lld is too large",
              (long long)p.rows, (long long)p.chans);
  g.tiles_n = static_cast<int>(tiles_n);
  constexpr bool kHalf = std::is_same_v<T, __half>;
  const uint32_t fmt = kHalf ? 0u : 1u;
  g.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (p.a_mn ? 1u << 15 : 0u) | (p.b_mn ? 1u << 16 : 0u) |
            (static_cast<uint32_t>(g.bn >> 3) << 17) | (static_cast<uint32_t>(kM >> 4) << 24);
  CUtensorMap ma, mb;
  if (encode(&ma, p.a, kHalf, P, p.a_mn ? 64 : KB, p.a_mn ? KB : kM, !p.a_mn && KB == 32) ||
      encode(&mb, p.b, kHalf, P, p.b_mn ? 64 : KB, p.b_mn ? KB : g.bn, !p.b_mn && KB == 32))
    return -1;
  auto kernel = linear_tc_kernel<T, P, KB>;
  PTB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  const int64_t tiles = static_cast<int64_t>(g.tiles_m) * g.tiles_n;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(g.split > 1 ? tiles * g.split : std::min<int64_t>(tiles, h->sms)));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = g.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  PTB_CUDA(cudaLaunchKernelEx(&cfg, kernel, ma, mb, g, h->gerr));
  count_launch();
  return 0;
}

}  // namespace

namespace ptb {

int64_t tc_plane_bytes(int dtype, int64_t rows, int64_t cols) {
  const int64_t ld = round_up(cols, 8);
  return round_up(rows * ld * 2 * (dtype == PT_B200_F32 ? 3 : 1), 256);
}

bool tc_direct(int dtype, const void *p, int64_t rows, int64_t ld) {
  return dtype != PT_B200_F32 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || ld % 8 == 0);
}

TcOperand tc_planes(void *p, int64_t rows, int64_t cols) {
  const int64_t ld = round_up(cols, 8);
  return TcOperand{p, rows, cols, ld, rows * ld};
}

TcOperand tc_tensor(const void *p, int64_t rows, int64_t cols, int64_t ld) {
  return TcOperand{p, rows, cols, rows == 1 ? round_up(cols, 8) : ld, 0};
}

int tc_pack(const pt_b200_ops *h, int dtype, const void *src, int64_t ld, const TcOperand &to, cudaStream_t st) {
  const PackArgs a{src, const_cast<void *>(to.p), to.rows, to.cols, ld, to.ld, to.plane};
  const int64_t blocks = std::min<int64_t>((to.rows * to.ld + 255) / 256, static_cast<int64_t>(h->sms) * 16);
  return with_dtype(dtype, [&](auto *z) -> int {
    pack_kernel<std::remove_pointer_t<decltype(z)>><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a);
    PTB_CUDA(cudaGetLastError());
    count_launch();
    return 0;
  });
}

int tc_product(const pt_b200_ops *h, int dtype, const TcProduct &p, cudaStream_t st) {
  switch (dtype) {
    case PT_B200_F32: return launch<float, 3, 32>(h, p, st);
    case PT_B200_BF16: return launch<__nv_bfloat16, 1, 64>(h, p, st);
    default: return launch<__half, 1, 64>(h, p, st);
  }
}

}  // namespace ptb
