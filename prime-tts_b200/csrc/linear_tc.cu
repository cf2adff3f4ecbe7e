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
// The tensor core's fp32 accumulator truncates each addition, which biases a long sum: fp16 gradients of
// weights over 262144 rows of one sign came out 2.1e-4 too small, over 4194304 rows 3.3e-3.  So an
// accumulator takes a chunk of k, and the epilogue warps add a tile's chunks in registers, rounding to
// nearest.
//
// bf16 and fp16 run as they are (one plane), 4096 of k a chunk: less than 256 x 2^-24 is lost, a thirtieth
// of fp16's rounding, and calls of up to 4096 of k, with one accumulator a tile, have a kernel without the
// sums in registers.  It costs nothing (65536 x 1024 x 1024 bf16 gradients 259 us, 278 before; with
// chunks of 1024, 16384 x 4096 x 4096 takes 354 us instead of 348).
//
// An fp32 operand is the sum of three bf16 planes (3 x 8 significant bits; the differences are exact),
// and the product is the six plane products that reach 2^-24 of it: a3 b1, a1 b3, a2 b2, a2 b1, a1 b2,
// a1 b1, smallest first, with a chunk of 64 of k.  The second plane is kept 2^7 and the third 2^14 times
// as large, because bf16 has fp32's exponents: unscaled, operands under 1e-33 lost their low planes (1e-36
// to an error of 2.7e-5).  The accumulator is taken times 2^-7 where the products go from one pair of
// scales to the next, which the MMA does on the way and in the same time (19434 x 192 x 768 54.2 us with
// and without).
//
// One CTA per SM walks its tiles: a TMA producer warp, an MMA warp, sixteen epilogue warps.  Two
// accumulators in TMEM let the epilogue of one tile run beside the next tile's MMAs.
//
// Large products run on CTA pairs (G = 2): one MMA of 256 channels over both SMs, each holding its
// 128 channels of A and half of the tile's rows of B, so that an SM reads and fetches half as much
// of B for the same arithmetic.  Products of few tiles run on single CTAs, and when there are
// fewer tiles than SMs a cluster of them shares a tile's k range: each leaves its part in its
// shared memory and adds a slice of the columns from all of them through distributed shared
// memory, in the order of the parts.
#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>

#include "drain.h"
#include "linear_tc.cuh"
#include "ptx.cuh"

using namespace ptb;

namespace ptb {
int tensor_map_encoder(PFN_cuTensorMapEncodeTiled_v12000 *fn);   // conv_tc.cu
}

namespace {

constexpr int kEpiWarps = 16;   // four to a quarter of the lanes: two left an epilogue of gelu and two stores latency-bound
constexpr int kFirstEpi = 3;
constexpr int kTcThreads = (kFirstEpi + kEpiWarps) * 32;   // warps 0 and 2 copy A and B, warp 1 MMA, the rest epilogue
constexpr int kM = 128;
constexpr uint32_t kTcWait = 1u << 21;   // tries of a wait inside a kernel that runs for milliseconds
constexpr int kMaxBn1 = 256, kMaxBn3 = 128;   // rows per tile; three planes' sums are in registers
constexpr int KB = 64;   // elements of k per stage: a 128-byte row
constexpr int kMaxStages = 10;
constexpr int kChunkStages = 64;   // one plane: stages that an accumulator takes at most
constexpr int kMaxSplit = 8;
constexpr int kSmemBudget = 217 * 1024;
constexpr int kSumLanes = 8;
constexpr int kSumBytes = kSumLanes * 33 * 4;
constexpr int kSmemBytes = kSmemBudget + 1024 + 512 + kSumBytes;

// t / d for 0 <= t < 2^31 as a multiplication: mul = ceil(2^(31 + s) / d) with 2^s >= d is off by
// less than 2^s / 2^31 of a quotient step, which t cannot make up.
struct Divide {
  uint32_t mul;
  int shift;
  explicit Divide(uint32_t d = 1) {
    int s = 0;
    while ((1u << s) < d) ++s;
    mul = static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + d - 1) / d);
    shift = 31 + s;
  }
  __device__ __forceinline__ int of(int t) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(t)) * mul) >> shift);
  }
};
constexpr int kBand = 16;

// One product of a launch.
struct TcOne {
  LinearEpi e;
  int64_t rows, chans;      // output rows (N side) and channels (M side)
  int kiters;               // k stages in all
  int per;                  // k stages of one of the CTAs that share a tile's k range
  int chunk;                // k stages of one accumulator
  int bn;                   // rows per tile
  int tiles_m, tiles_n;     // channel tiles, row tiles
  Divide by_band;           // by the tiles of a band
  Divide by_last;           // by the channel tiles of the last band, where it is not a whole one
  uint32_t idesc;
  bool a_mn, b_mn;
};
// One product, or two (the gradient's).  Worker w of W (a CTA, a pair, a cluster) takes tiles w, w + W,
// ... of the first product, whose tiles are the longer ones; then all workers take the second's in
// turns, but after `both` turns only those that had one tile less of the first, from `late` on.
constexpr int kMaxProducts = 2;
struct TcArgs {
  TcOne p[kMaxProducts];
  int tiles[kMaxProducts];
  int both, late;
  int split;                // CTAs that share a tile's k range (the cluster)
  int stages;
  uint32_t stage_bytes;
  uint32_t acc_cols;        // TMEM columns from one accumulator to the next, a power of two
  bool beside;              // needs nothing of the kernel launched right before it
  ColumnSums sums;          // done beside the first tile, or parts = 0
};
struct TcMaps {
  CUtensorMap a[kMaxProducts], b[kMaxProducts];
};

// ---- the same steps for one CTA (G = 1) and for a pair (G = 2, issued by its rank 0)
// Descriptors come as their low words (the address moves, 16 bytes a step) and the constant high
// word.  kFirst starts the accumulator where `keep` is 0, kShift adds to it after taking it times
// 2^-kPlaneShift, any other MMA adds to it.
enum class Acc { kFirst, kShift, kAdd };
template <int G, Acc ACC>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                        uint32_t keep) {
#define PTB_MMA(group, pred, shift)                                                                       \
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"                                               \
               "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t" pred                                   \
               "tcgen05.mma.cta_group::" group ".kind::f16 [%0], a, b, %4, p" shift ";\n\t}" ::"r"(d_tmem), \
               "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(keep), "n"(kPlaneShift)                     \
               : "memory")
#define PTB_KEEP "setp.ne.b32 p, %5, 0;\n\t"
#define PTB_ALWAYS "setp.ne.b32 p, 1, 0;\n\t"
  if constexpr (G == 1 && ACC == Acc::kFirst) PTB_MMA("1", PTB_KEEP, "");
  if constexpr (G == 1 && ACC == Acc::kShift) PTB_MMA("1", PTB_ALWAYS, ", %6");
  if constexpr (G == 1 && ACC == Acc::kAdd) PTB_MMA("1", PTB_ALWAYS, "");
  if constexpr (G == 2 && ACC == Acc::kFirst) PTB_MMA("2", PTB_KEEP, "");
  if constexpr (G == 2 && ACC == Acc::kShift) PTB_MMA("2", PTB_ALWAYS, ", %6");
  if constexpr (G == 2 && ACC == Acc::kAdd) PTB_MMA("2", PTB_ALWAYS, "");
#undef PTB_KEEP
#undef PTB_ALWAYS
#undef PTB_MMA
}
// Arrives on the barrier at this offset, of both CTAs of a pair, once the MMAs so far are done.
template <int G>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (G == 1)
    mma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
template <int G>
__device__ __forceinline__ void alloc(uint32_t slot, uint32_t cols) {
  if constexpr (G == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int G>
__device__ __forceinline__ void dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (G == 1)
    tmem_dealloc(taddr, cols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// A tile into this CTA's shared memory; `bar` may be the other CTA's of the pair.
template <int G>
__device__ __forceinline__ void load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2) {
  if constexpr (G == 1)
    tma_load_3d(dst, map, bar, c0, c1, c2);
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// True in one lane of the warp.  The roles below run with all lanes, so that their loop state is
// the same in every lane and stays in uniform registers, and only the copies and MMAs themselves
// are issued by one: with the whole loop inside one lane's branch, an MMA took 140 clocks to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
// The same value in every lane, and known to be.
template <class V>
__device__ __forceinline__ V uniform(V v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ uint32_t in_rank0(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// An accumulator is free again.  Only TMEM loads, already waited for, come before it: no memory has
// to be released, and a cluster-wide release took 1100 to 3800 clocks of every chunk.
template <int G>
__device__ __forceinline__ void arrive(uint32_t bar) {
  if constexpr (G == 1)
    mbar_arrive(bar);
  else
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Shared-memory descriptors.  K-major: rows of KB = 64 elements (128 bytes, swizzled by as much),
// atoms of 8 rows one after another.  MN-major: blocks of 64 elements (128 bytes, swizzled) x KB
// rows of k; `lead` bytes from one block of 64 to the next, 8 rows of k to an atom.
__device__ __forceinline__ uint32_t sdesc_lo(uint32_t saddr, uint32_t lead) {
  return ((saddr >> 4) & 0x3FFFu) | (((lead >> 4) & 0x3FFFu) << 16);
}
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);   // atom, version, 128-byte swizzle

// Tile t of the walk: channel tiles fastest inside bands of kBand, so that concurrent CTAs share
// both operands through L2.
__device__ __forceinline__ void tile_at(const TcOne &g, int t, int *tm, int *tn) {
  const int band = g.by_band.of(t);
  const int in = t - band * kBand * g.tiles_n;
  const bool last = (band + 1) * kBand > g.tiles_m;
  const int across = last ? g.by_last.of(in) : in / kBand;
  *tm = band * kBand + in - across * (last ? g.tiles_m - band * kBand : kBand);
  *tn = across;
}

// Sixteen results of one channel, rows row0 .. row0 + 15: bias, activation, residual, store.
struct ActOnAll {
  float (&v)[16];
  float slope;
  template <int ACT>
  __device__ __forceinline__ void operator()() const {
    if constexpr (ACT != PT_B200_ACT_NONE)
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const float2 o = act_value<ACT>(make_float2(v[j], v[j + 1]), slope);
        v[j] = o.x, v[j + 1] = o.y;
      }
  }
};
template <class T>
__device__ __forceinline__ void emit16(const LinearEpi &e, float (&v)[16], int64_t chan, int64_t row0, int n,
                                       float bias) {
  float r[16];
  if (e.residual) {
    const T *p = static_cast<const T *>(e.residual) + row0 * e.ldr + chan;
#pragma unroll
    for (int j = 0; j < 16; ++j, p += e.ldr) r[j] = j < n ? to_f32(*p) : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] += bias;
  if (e.pre) {
    T *p = static_cast<T *>(e.pre) + row0 * e.ldp + chan;
#pragma unroll
    for (int j = 0; j < 16; ++j, p += e.ldp)
      if (j < n) *p = from_f32<T>(v[j]);
  }
  with_act(e.act, ActOnAll{v, e.slope});
  if (e.residual) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += r[j];
  }
  T *p = static_cast<T *>(e.y) + row0 * e.ldy + chan;
#pragma unroll
  for (int j = 0; j < 16; ++j, p += e.ldy)
    if (j < n) *p = from_f32<T>(v[j]);
}

// Waits for the copies that two producers have issued.  (Not inlined: nothing is live where it is called, and
// no call that ends as it should comes here.)
__device__ __noinline__ void drain_copies(uint32_t full, int stages, int a, int b, int lane, uint32_t *gerr) {
  const Drain d = drain_of(a, b, stages);
  for (int i = d.begin; i < d.end; ++i) {
    const uint32_t bar = full + 8u * (i % stages);
    if (i >= d.matched && lane == 0) mbar_arrive(bar);
    __syncwarp();
    uint32_t it = 0;
    while (!mbar_try_wait(bar, fill_parity(i, stages)) && ++it < kTcWait) {
    }
    if (it >= kTcWait && lane == 0) atomicOr(gerr, ERR_WAIT_DRAIN);
  }
}

// G CTAs to a tile, P planes per operand; kChunks: a tile's k may take several accumulators.
template <class T, int G, int P, bool kChunks>
__global__ void __launch_bounds__(kTcThreads, 1)
    linear_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcArgs args, uint32_t *gerr) {
  namespace cg = cooperative_groups;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *gbase = smem_raw + (base - raw);
  constexpr uint32_t a_plane = kM * KB * 2;
  const uint32_t stage_bytes = args.stage_bytes, acc_cols = args.acc_cols;
  const uint32_t bar0 = base + kSmemBudget;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  // accumulators: two, or (three planes) two for each team of epilogue warps
  constexpr int kTeams = P == 1 ? 1 : 2, kBuffers = 2 * kTeams;
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kMaxStages + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kMaxStages + 4 + b); };   // rank 0's counts
  const uint32_t drain = bar0 + 8u * (2 * kMaxStages + 8);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(gbase + kSmemBudget + 8 * (2 * kMaxStages + 9));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *issued_of = reinterpret_cast<int *>(tmem_slot + 2);   // stages that the producers have copied, B's and A's

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t tmem_cols = kBuffers * acc_cols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < args.stages; ++s) {
      mbar_init(full(s), 2);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < kBuffers; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), G * kEpiWarps / kTeams);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&maps.a[0]);
    prefetch_tmap(&maps.b[0]);
  }
  if (warp == 1) {
    alloc<G>(smem_u32(tmem_slot), tmem_cols);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (G == 2) cg::this_cluster().sync();   // the other CTA's barriers are ready too
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  // What follows reads and writes global memory: after the kernels before this one.
  if (!args.beside) wait_for_previous();
  let_next_start();

  // The CTAs of a cluster work on a tile together: the pair, or those that share its k range.
  int rank, first, step;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(first));
  asm("mov.u32 %0, %%nclusterid.x;" : "=r"(step));
  const int pair_rank = G == 2 ? rank : 0;
  const int k_rank = G == 2 ? 0 : rank;
  // the n-th tile of this worker: its product, its place, and this CTA's stages of k
  struct Tile {
    const TcOne &g;
    int which, tm, tn, k_lo, k_hi;
  };
  const int longs = first < args.tiles[0] ? (args.tiles[0] - first - 1) / step + 1 : 0;
  auto place = [&](int n, int *which) -> int {   // -1: no more
    *which = n >= longs;
    if (!*which) return first + n * step;
    const int turn = n - longs;
    if (turn >= args.both && first < args.late) return -1;
    const int t = turn < args.both ? turn * step + first
                                   : args.both * step + (turn - args.both) * (step - args.late) + first - args.late;
    return t < args.tiles[1] ? t : -1;
  };
  auto tile = [&](int t, int which) -> Tile {
    const TcOne &g = args.p[which];
    int tm, tn;
    tile_at(g, t, &tm, &tn);
    const int k_lo = k_rank * g.per;
    return Tile{g, which, tm, tn, k_lo, min(k_lo + g.per, g.kiters)};
  };

  // (known to the compiler where it is one stage: read from the arguments, 65536 x 192 x 192 gradients of three
  // planes took 198 us instead of 177)
  auto chunk_of = [](const TcOne &g) { return P == 1 ? g.chunk : 1; };

  if (warp == 0 || warp == 2) {
    // ---------------- TMA producers: A in warp 0, B in warp 2 (a copy takes 80 to 120 clocks to issue)
    const bool is_a = warp == 0;
    const bool one = elect_one();
    int s = 0, issued = 0;
    uint32_t phase = 0, a0 = is_a ? base : base + P * a_plane;
    // a pair's copies all count on rank 0's barrier, where the MMAs are issued
    const uint32_t bar0_of = G == 1 ? full(0) : in_rank0(full(0));
    bool ok = true;
    for (int n = 0, t, which; ok && (t = place(n, &which)) >= 0; ++n) {
      const Tile at_tile = tile(t, which);
      const TcOne &g = at_tile.g;
      const CUtensorMap *map = is_a ? &maps.a[which] : &maps.b[which];
      const int b_rows = g.bn / G;                     // rows of B in this CTA
      const uint32_t plane = is_a ? a_plane : static_cast<uint32_t>(b_rows) * KB * 2;
      const int chan0 = uniform((at_tile.tm * G + pair_rank) * kM);
      const int row0 = uniform(at_tile.tn * g.bn + pair_rank * b_rows);
      for (int k = at_tile.k_lo; k < at_tile.k_hi; ++k) {
        if (issued >= args.stages && !mbar_wait(empty(s), phase ^ 1u, abort_flag, gerr, ERR_WAIT_EMPTY, kTcWait)) {
          ok = false;
          break;
        }
        const uint32_t bar = uniform(bar0_of + 8u * s), own = uniform(full(s));
        const int ku = uniform(k * KB);
        uint32_t at = uniform(a0);
        if (one) {
          if (pair_rank == 0) mbar_expect_tx(own, G * P * plane);
          if (is_a) {
#pragma unroll
            for (int p = 0; p < P; ++p, at += a_plane) {
              if (g.a_mn) {
#pragma unroll
                for (int i = 0; i < kM / 64; ++i) load<G>(at + i * KB * 128, map, bar, chan0 + i * 64, ku, p);
              } else {
                load<G>(at, map, bar, ku, chan0, p);
              }
            }
          } else {
#pragma unroll
            for (int p = 0; p < P; ++p, at += plane) {
              if (g.b_mn) {
                for (int i = 0; i < b_rows / 64; ++i) load<G>(at + i * KB * 128, map, bar, row0 + i * 64, ku, p);
              } else {
                load<G>(at, map, bar, ku, row0, p);
              }
            }
          }
        }
        ++issued;
        a0 += stage_bytes;
        if (++s == args.stages) s = 0, phase ^= 1u, a0 -= args.stages * stage_bytes;
      }
    }
    if (lane == 0) issued_of[is_a] = issued;
    if (pair_rank == 0) asm volatile("bar.arrive 2, 96;" ::: "memory");   // both producers are through: for the MMA warp
  } else if (warp == 1) {
    if (pair_rank == 0) {
      // ---------------- MMA issuer
      const bool one = elect_one();
      int s = 0, turn = 0, units[2] = {0, 0};   // accumulators given to each team so far
      uint32_t phase = 0, at = 0;    // `at`: the stage's place, in the descriptors' 16 bytes
      bool ok = true;
      for (int n = 0, t, which; ok && (t = place(n, &which)) >= 0; ++n) {
        const Tile at_tile = tile(t, which);
        const TcOne &g = at_tile.g;
        const uint32_t b_plane = static_cast<uint32_t>(g.bn / G) * KB * 2;
        const uint32_t a_adv = g.a_mn ? 2048u >> 4 : 32u >> 4;     // 16 elements of k further on
        const uint32_t b_adv = g.b_mn ? 2048u >> 4 : 32u >> 4;
        const uint32_t da0 = sdesc_lo(base, g.a_mn ? KB * 128 : 16);
        const uint32_t db0 = sdesc_lo(base + P * a_plane, g.b_mn ? KB * 128 : 16);
        const int k_hi = at_tile.k_hi;
        const int team = P == 1 ? 0 : turn++ & 1;
        int unit = team ? units[1] : units[0];
        for (int k = at_tile.k_lo; k < k_hi && ok; ++unit) {
          const int b = 2 * team + (unit & 1);
          if (unit >= 2 && !mbar_wait(acc_empty(b), ((unit >> 1) & 1) ^ 1u, abort_flag, gerr, ERR_WAIT_ACC, kTcWait)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = uniform(tmem + b * acc_cols);
          const int k_end = kChunks ? min(k + chunk_of(g), k_hi) : k_hi;
          uint32_t accumulate = 0;
          for (; k < k_end; ++k) {
            if (!mbar_wait(full(s), phase, abort_flag, gerr, ERR_WAIT_FULL, kTcWait)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t here = uniform(at), first_of = uniform(accumulate), free_bar = uniform(empty(s));
            if (one) {
#pragma unroll
              for (int q = 0; q < (P == 1 ? 1 : 6); ++q) {
                constexpr int kPa[6] = {2, 0, 1, 1, 0, 0}, kPb[6] = {0, 2, 1, 0, 1, 0};
                const uint32_t da = da0 + here + (P == 1 ? 0 : kPa[q]) * (a_plane >> 4);
                const uint32_t db = db0 + here + (P == 1 ? 0 : kPb[q]) * (b_plane >> 4);
                if (q == 0)
                  mma_f16<G, Acc::kFirst>(d, da, db, kDescHi, g.idesc, first_of);
                else if (kPa[q] + kPb[q] < kPa[q - 1] + kPb[q - 1])   // the next planes: what is there is shifted
                  mma_f16<G, Acc::kShift>(d, da, db, kDescHi, g.idesc, 1);
                else
                  mma_f16<G, Acc::kAdd>(d, da, db, kDescHi, g.idesc, 1);
#pragma unroll
                for (int i = 1; i < KB / 16; ++i)
                  mma_f16<G, Acc::kAdd>(d, da + i * a_adv, db + i * b_adv, kDescHi, g.idesc, 1);
              }
              commit<G>(free_bar);
            }
            accumulate = 1;
            at += stage_bytes >> 4;
            if (++s == args.stages) s = 0, phase ^= 1u, at = 0;
          }
          if (ok && one) commit<G>(acc_full(b));
        }
        (team ? units[1] : units[0]) = unit;
      }
      asm volatile("bar.sync 2, 96;" ::: "memory");
      if (!ok) {
        // copies in flight must land before shared memory is given up, whichever producer issued them (a
        // pair's count on rank 0's barriers; rank 1 stops only after a wait of its own), and MMAs already
        // issued must finish before TMEM is
        drain_copies(full(0), args.stages, issued_of[1], issued_of[0], lane, gerr);
        if (one) commit<G>(drain);
        uint32_t it = 0;
        while (!mbar_try_wait(drain, 0) && ++it < kTcWait) {
        }
        if (it >= kTcWait && one) atomicOr(gerr, ERR_WAIT_DRAIN);
      }
    }
  } else {
    // ---------------- epilogue warps: lanes 32 (warp % 4) .. + 31, every fourth block of 16 columns
    const int part_of = warp - kFirstEpi, quad = warp & 3, team = P == 1 ? 0 : part_of >> 3;
    const uint32_t tl = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    if (args.sums.parts > 0 && warp < kFirstEpi + kSumLanes) {   // column sums, 32 columns at a time, while the first tile's products run
      float *red = reinterpret_cast<float *>(gbase + kSmemBudget + 512);
      const int row = warp - kFirstEpi;
      for (int64_t c0 = blockIdx.x * 32; c0 < args.sums.n; c0 += gridDim.x * 32) {
        float v = 0.0f;
        if (c0 + lane < args.sums.n) v = lane_sum(args.sums.part + c0 + lane, row, args.sums.parts, kSumLanes, args.sums.n);
        red[row * 33 + lane] = v;
        asm volatile("bar.sync 1, %0;" ::"n"(kSumLanes * 32) : "memory");
        if (row == 0 && c0 + lane < args.sums.n) {
          v = 0.0f;
          for (int i = 0; i < kSumLanes; ++i) v += red[i * 33 + lane];
          static_cast<T *>(args.sums.out)[c0 + lane] = from_f32<T>(v);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kSumLanes * 32) : "memory");
      }
    }
    int unit = 0, turn = 0;
    bool ok = true;
    for (int n = 0, t, which; ok && (t = place(n, &which)) >= 0; ++n) {
      const Tile at_tile = tile(t, which);
      const TcOne &g = at_tile.g;
      const int64_t chan = static_cast<int64_t>(at_tile.tm * G + pair_rank) * kM + quad * 32 + lane;
      const int64_t row0 = static_cast<int64_t>(at_tile.tn) * g.bn;
      const float bias = g.e.bias && chan < g.chans ? to_f32(static_cast<const T *>(g.e.bias)[chan]) : 0.0f;
      float *part = reinterpret_cast<float *>(gbase);   // split: [bn][128] of this CTA's part
      if constexpr (!kChunks) {
        const int b = unit & 1;
        if (!mbar_wait(acc_full(b), (unit >> 1) & 1, abort_flag, gerr, ERR_WAIT_ACC, kTcWait)) break;
        tc_fence_after();
        for (int c = (part_of >> 2) * 16; c < g.bn; c += 64) {
          float v[16];
          tmem_ld16(tl + b * acc_cols + c, v);
          if (args.split > 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(c + j) * kM + quad * 32 + lane] = v[j];
          } else {
            const int n = static_cast<int>(min(static_cast<int64_t>(16), g.rows - row0 - c));
            if (chan < g.chans && n > 0) emit16<T>(g.e, v, chan, row0 + c, n, bias);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive<G>(G == 1 ? acc_empty(b) : in_rank0(acc_empty(b)));
        ++unit;
      } else {
        // Three planes: two teams of eight warps take turns at the tiles, one adds up the chunks of a
        // tile while the other still stores the one before (19434 x 192 x 768 spent 4700 of a tile's
        // 7900 clocks on its stores with one team).
        if (kTeams == 2 && turn++ % 2 != team) continue;
        // a warp's columns: blocks of 16, every kGroups-th
        constexpr int kGroups = kEpiWarps / kTeams / 4, kBlocks = (P == 1 ? kMaxBn1 : kMaxBn3) / (16 * kGroups);
        const int c0 = (part_of / 4 % kGroups) * 16;
        float acc[kBlocks][16];
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[i][j] = P == 1 ? -0.0f : 0.0f;   // (-0 leaves a single chunk's bits as they are)
        for (int k = at_tile.k_lo; k < at_tile.k_hi && ok; k += chunk_of(g), ++unit) {
          const int b = 2 * team + (unit & 1);
          if (!mbar_wait(acc_full(b), (unit >> 1) & 1, abort_flag, gerr, ERR_WAIT_ACC, kTcWait)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) {
            if (c0 + i * 16 * kGroups < g.bn) {
              float v[16];
              tmem_ld16(tl + b * acc_cols + c0 + i * 16 * kGroups, v);
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[i][j] += v[j];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive<G>(G == 1 ? acc_empty(b) : in_rank0(acc_empty(b)));
        }
        if (!ok) break;
        if (args.split > 1) {
          // the stages still hold operands of the last chunk until its MMAs are done, which the
          // last accumulator's arrival says
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) {
            const int c = c0 + i * 16 * kGroups;
            if (c < g.bn)
#pragma unroll
              for (int j = 0; j < 16; ++j) part[(c + j) * kM + quad * 32 + lane] = acc[i][j];
          }
        } else {
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) {
            const int c = c0 + i * 16 * kGroups;
            const int n = static_cast<int>(min(static_cast<int64_t>(16), g.rows - row0 - c));
            if (c < g.bn && chan < g.chans && n > 0) emit16<T>(g.e, acc[i], chan, row0 + c, n, bias);
          }
        }
      }
    }
  }
  __syncwarp();
  if (G == 1 && args.split > 1) {
    // ---------------- one tile per cluster: add the parts, a slice of the rows per CTA
    auto cluster = cg::this_cluster();
    cluster.sync();
    if (warp >= kFirstEpi && !*abort_flag) {
      const int quad = warp & 3, half = (warp - kFirstEpi) >> 2, split = args.split;
      const Tile at_tile = tile(first, 0);
      const TcOne &g = at_tile.g;
      const int64_t chan = static_cast<int64_t>(at_tile.tm) * kM + quad * 32 + lane;
      float *part = reinterpret_cast<float *>(gbase);
      const int width = g.bn / split;
      const float *from[kMaxSplit];
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        from[r] = cluster.map_shared_rank(part, r < split ? r : 0) + quad * 32 + lane;
      for (int c = rank * width + half; c < (rank + 1) * width; c += 4) {
        const int64_t row = static_cast<int64_t>(at_tile.tn) * g.bn + c;
        float got[kMaxSplit], v = 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r) got[r] = r < split ? from[r][c * kM] : 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r) v += got[r];
        if (chan < g.chans && row < g.rows) linear_store<T>(g.e, row, chan, v);
      }
    }
    cluster.sync();   // no CTA leaves while another still reads its part
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (G == 2) cg::this_cluster().sync();   // nor while the pair's MMAs or arrivals reach it
  if (warp == 1) {
    tc_fence_after();
    dealloc<G>(tmem, tmem_cols);
  }
  // a kernel that ran beside the one before it ends after it: the next may wait for this one alone
  if (args.beside) wait_for_previous();
}

// ------------------------------------------------------------------------------ operand passes
constexpr int kPrepBlock = 256;
constexpr int kPrepRows = 1;   // rows a thread has in flight: 2 and 4 cost blocks of an SM and were 8 to 40% slower
constexpr int kPrepPerSm = 4;  // blocks of a pass that run on one SM at once, and that it is cut into

template <class T>
struct alignas(16) Eight {
  T v[8];
};
template <class T>
__device__ __forceinline__ void load8(const T *p, int n, bool vec, Eight<T> *o) {
  if (vec) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / V; ++i)
      *reinterpret_cast<uint4 *>(o->v + i * V) = __ldcs(reinterpret_cast<const uint4 *>(p + i * V));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o->v[i] = i < n ? p[i] : from_f32<T>(0.0f);
  }
}

// One thread's rows of a job: eight columns of every `step`-th row from r0.
template <class T>
struct PrepRows {
  const PrepJob &a;
  int64_t c, r0, step;
  int n;
  float2 (&sum)[4];
  template <int ACT>
  __device__ __forceinline__ void operator()() const {
    for (int64_t r1 = r0; r1 < a.rows; r1 += kPrepRows * step) {
      Eight<T> s[kPrepRows], p[kPrepRows];
#pragma unroll
      for (int u = 0; u < kPrepRows; ++u) {
        const int64_t r = r1 + u * step;
        if (r < a.rows) {
          load8(static_cast<const T *>(a.src) + r * a.ld + c, n, a.vec, &s[u]);
          if constexpr (ACT != PT_B200_ACT_NONE)
            load8(static_cast<const T *>(a.pre) + r * a.ldp + c, n, a.vec, &p[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < kPrepRows; ++u) {
        const int64_t r = r1 + u * step;
        if (r >= a.rows) break;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          float2 t = make_float2(to_f32(s[u].v[i]), to_f32(s[u].v[i + 1]));
          if constexpr (ACT != PT_B200_ACT_NONE)
            t = mul2(t, act_grad<ACT>(make_float2(to_f32(p[u].v[i]), to_f32(p[u].v[i + 1])), a.slope));
          sum[i / 2] = add2(sum[i / 2], t);
          d[i] = t.x, d[i + 1] = t.y;
        }
        if (!a.dst) continue;
        if constexpr (sizeof(T) == 4) {
          Pack<__nv_bfloat16, 8> o[3];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            __nv_bfloat16 q[3];
            split3(d[i], q);
            o[0].v[i] = q[0];
            o[1].v[i] = q[1];
            o[2].v[i] = q[2];
          }
#pragma unroll
          for (int i = 0; i < 3; ++i)
            *reinterpret_cast<Pack<__nv_bfloat16, 8> *>(static_cast<__nv_bfloat16 *>(a.dst) + i * a.plane +
                                                        r * a.ldd + c) = o[i];
        } else {
          // rounded to the operands' type for the products; the sums take the fp32 value
          Pack<T, 8> o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o.v[i] = from_f32<T>(d[i]);
          *reinterpret_cast<Pack<T, 8> *>(static_cast<T *>(a.dst) + r * a.ldd + c) = o;
        }
      }
    }
  }
};

// Bound by HBM: src and pre are read once and dst is written once, 16 bytes a thread at a time
// where rows are aligned.
template <class T>
__global__ void __launch_bounds__(kPrepBlock, kPrepPerSm) prep_kernel(const __grid_constant__ PrepJobs jobs) {
  __shared__ __align__(8) float red[kPrepBlock * 8];
  let_next_start();
  int job = 0, block = blockIdx.x;
#pragma unroll
  for (int i = 0; i < kMaxJobs - 1; ++i)
    if (static_cast<int>(blockIdx.x) >= jobs.end[i]) job = i + 1, block = blockIdx.x - jobs.end[i];
  const PrepJob &a = jobs.j[job];
  const int tx = threadIdx.x & (a.lanes - 1), ty = threadIdx.x / a.lanes, height = kPrepBlock / a.lanes;
  const int cb = block % a.col_blocks, rb = block / a.col_blocks;
  const int64_t c = (static_cast<int64_t>(cb) * a.lanes + tx) * 8;
  const int n = static_cast<int>(min(static_cast<int64_t>(8), a.cols - c));
  float2 sum[4] = {};
  if (n > 0)
    with_act(a.act, PrepRows<T>{a, c, static_cast<int64_t>(rb) * height + ty,
                                static_cast<int64_t>(a.row_blocks) * height, n, sum});
  if (!a.part) return;
  // the block's row lanes, added in order
  const int width = a.lanes * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<float2 *>(red + ty * width + tx * 8 + 2 * i) = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < width; i += kPrepBlock) {
    const int64_t col = static_cast<int64_t>(cb) * width + i;
    if (col >= a.cols) break;
    float v = 0.0f;
    for (int k = 0; k < height; ++k) v += red[k * width + i];
    a.part[static_cast<int64_t>(rb) * a.cols + col] = v;
  }
}

int encode(CUtensorMap *m, const TcOperand &o, bool half, int planes, int box_inner, int box_outer) {
  PFN_cuTensorMapEncodeTiled_v12000 enc;
  if (tensor_map_encoder(&enc)) return -1;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(planes > 1 ? o.plane * 2 : 16)};
  cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                         const_cast<void *>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  PTB_REQUIRE(r == CUDA_SUCCESS, "pt_b200: operand tensor map encode failed (%d)", (int)r);
  return 0;
}

// CTAs to a tile, rows per tile and k split: the cheapest of the candidates by a count of SM
// clocks, whose figures are measurements (B200, clocks read in the kernel at 64 of k a stage):
//   - an MMA of 16 of k takes bn / 2 clocks, or what its operands take to leave shared memory at
//     128 bytes a clock (4 KB of A, and B's rows of this CTA), next to the copies that fill it;
//   - a stage's bytes arrive at about 75 a clock (the L2's rate when all SMs ask: bf16 pairs of
//     128 rows 319 clocks a stage, of 224 rows 398), and no stage takes less than 330;
//   - a tile starts after 2800 and leaves after 300 + 15 bn, which the next tile hides;
//   - parts of a split tile are exchanged in 3500 + 4 bn.
// The clusters of a split must fit the GPU at once.
inline int k_stages(int64_t k) { return static_cast<int>((k + KB - 1) / KB); }
struct Shape {
  int group, bn, split;
  double clocks;   // of the call, and of one tile in a walk
  double tile;
};
Shape pick_shape(const pt_b200_ops *h, int64_t rows, int64_t chans, int kiters, int planes, bool b_mn) {
  Shape best{0, 0, 1, 0, 0};
  const int products = planes == 1 ? 1 : 6;
  for (int group : {1, 2}) {
    const int64_t tm = (chans + group * kM - 1) / (group * kM);
    for (int bn = 16; bn <= (planes == 1 ? kMaxBn1 : kMaxBn3); bn += 16) {
      // an MN-major tile is made of blocks of 64; accumulators of a pair start at 32 rows
      if ((b_mn && bn % (64 * group)) || (group == 2 && bn % 32)) continue;
      const double bytes = planes * KB * 2.0 * (kM + bn / group);
      if (2 * bytes > kSmemBudget) continue;   // two stages at least
      const int mmas = products * (KB / 16);
      const double stage = std::max(std::max(mmas * bn / 2.0, mmas * (32 + bn / (4.0 * group)) + bytes * 0.6 / 128),
                                    std::max(bytes / 75, 330.0));
      const double leave = 300 + 15.0 * bn;
      const int64_t tiles = tm * ((rows + bn - 1) / bn);
      for (int split = 1, log = 0; split <= kMaxSplit; split *= 2, ++log) {
        const int per = (kiters + split - 1) / split;
        if (split > 1 && (group == 2 || (split - 1) * per >= kiters || tiles > h->clusters[log])) continue;
        const int64_t at_once = group == 2 ? h->clusters[1] : h->clusters[log];
        const int64_t waves = (tiles + at_once - 1) / at_once;
        const double cost = 2800 + waves * std::max(per * stage, leave) + leave + (split > 1 ? 3500 + 4.0 * bn : 0);
        if (!best.bn || cost < best.clocks) best = Shape{group, bn, split, cost, std::max(per * stage, leave)};
      }
    }
  }
  return best;
}

template <class T, int P>
auto *tc_kernel(int group, bool chunks) {
  if constexpr (P == 3)
    return group == 1 ? linear_tc_kernel<T, 1, P, true> : linear_tc_kernel<T, 2, P, true>;
  else
    return chunks ? (group == 1 ? linear_tc_kernel<T, 1, P, true> : linear_tc_kernel<T, 2, P, true>)
                  : (group == 1 ? linear_tc_kernel<T, 1, P, false> : linear_tc_kernel<T, 2, P, false>);
}

template <class T, int P>
int launch(const pt_b200_ops *h, const TcProduct *products, const Shape *shapes, int count, const ColumnSums &sums,
           bool early, bool beside, int most, cudaStream_t st) {
  constexpr bool kHalf = std::is_same_v<T, __half>;
  const int G = shapes[0].group;
  TcArgs a{};
  TcMaps maps;
  a.sums = sums;
  a.beside = beside;
  a.split = shapes[0].split;
  a.acc_cols = 16;
  bool chunks = P == 3;
  for (int i = 0; i < count; ++i) {
    const TcProduct &p = products[i];
    TcOne &g = a.p[i];
    g.e = p.e;
    g.rows = p.rows;
    g.chans = p.chans;
    g.a_mn = p.a_mn;
    g.b_mn = p.b_mn;
    g.kiters = k_stages(p.k);
    g.bn = shapes[i].bn;
    g.per = (g.kiters + a.split - 1) / a.split;
    g.chunk = P == 1 ? kChunkStages : 1;
    chunks = chunks || g.per > g.chunk;
    g.tiles_m = static_cast<int>((p.chans + G * kM - 1) / (G * kM));
    const int64_t tiles_n = (p.rows + g.bn - 1) / g.bn;
    PTB_REQUIRE(tiles_n * g.tiles_m < (int64_t(1) << 29) && tiles_n < (int64_t(1) << 26),
                "pt_b200: product of %lld x %lld is too large",
                (long long)p.rows, (long long)p.chans);
    g.tiles_n = static_cast<int>(tiles_n);
    g.by_band = Divide(static_cast<uint32_t>(kBand * g.tiles_n));
    g.by_last = Divide(g.tiles_m % kBand ? g.tiles_m % kBand : kBand);
    const uint32_t fmt = kHalf ? 0u : 1u;
    g.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (p.a_mn ? 1u << 15 : 0u) | (p.b_mn ? 1u << 16 : 0u) |
              (static_cast<uint32_t>(g.bn >> 3) << 17) | (static_cast<uint32_t>(G * kM >> 4) << 24);
    if (encode(&maps.a[i], p.a, kHalf, P, p.a_mn ? 64 : KB, p.a_mn ? KB : kM) ||
        encode(&maps.b[i], p.b, kHalf, P, p.b_mn ? 64 : KB, p.b_mn ? KB : g.bn / G))
      return -1;
    a.stage_bytes = std::max(a.stage_bytes, static_cast<uint32_t>(round_up(P * (kM + g.bn / G) * KB * 2, 1024)));
    while (a.acc_cols < static_cast<uint32_t>(g.bn)) a.acc_cols *= 2;
    a.tiles[i] = g.tiles_m * g.tiles_n;
  }
  if (count == 1) maps.a[1] = maps.a[0], maps.b[1] = maps.b[0];
  a.stages = std::min<int>(kMaxStages, kSmemBudget / a.stage_bytes);
  auto *kernel = tc_kernel<T, P>(G, chunks);
  const int group = G * a.split;
  const int all = a.tiles[0] + a.tiles[1];
  const int workers = a.split > 1 ? all : std::min({all, most, group == 1 ? h->clusters[0] : h->clusters[1]});
  // the turns that all workers take part in: those that end the call soonest
  const int busy = a.tiles[0] % workers;   // workers with one long tile more
  a.both = a.tiles[1];
  if (count == 2 && busy) {
    const double c0 = a.p[0].kiters * static_cast<double>(a.p[0].bn), c1 = a.p[1].kiters * static_cast<double>(a.p[1].bn);
    double best = 0;
    for (int both = 0; both <= (a.tiles[1] + workers - 1) / workers; ++both) {
      const int left = std::max(0, a.tiles[1] - both * workers);
      const int more = (left + workers - busy - 1) / (workers - busy);
      const double end = std::max(c0 + both * c1, (both + more) * c1);
      if (both == 0 || end < best) best = end, a.both = both;
    }
    a.late = busy;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(group * workers));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = group;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 2 : 1;
  PTB_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps, a, h->gerr));
  count_launch();
  return 0;
}

template <class T, int P>
int launch_products(const pt_b200_ops *h, const TcProduct *p, int count, ColumnSums sums, bool early,
                    cudaStream_t st) {
  Shape sh[kMaxProducts];
  for (int i = 0; i < count; ++i) sh[i] = pick_shape(h, p[i].rows, p[i].chans, k_stages(p[i].k), P, p[i].b_mn);
  // products of one kind of cluster share a launch (a split one only while its clusters all fit); the
  // shape of each is its own, so that its sums are the same alone and in company
  if (count == 2 && sh[0].group == sh[1].group && sh[0].split == 1 && sh[1].split == 1) {
    const bool swap = k_stages(p[1].k) * static_cast<double>(sh[1].bn) > k_stages(p[0].k) * static_cast<double>(sh[0].bn);
    const TcProduct two[2] = {p[swap], p[!swap]};   // longer tiles first
    const Shape shapes[2] = {sh[swap], sh[!swap]};
    return launch<T, P>(h, two, shapes, 2, sums, early, false, INT_MAX, st);
  }
  // Otherwise one after the other, which start together where there is room: the second needs the same
  // passes as the first and nothing of it.  A split product leaves SMs free, so it goes first, and the
  // other keeps to those SMs if it is done there in the meantime.
  const bool swap = count == 2 && sh[1].split > sh[0].split;
  for (int i = 0; i < count; ++i) {
    const int at = swap ? 1 - i : i;
    int most = INT_MAX;
    if (i == 1 && sh[1 - at].split > 1 && sh[at].split == 1) {
      const TcProduct &q = p[1 - at], &mine = p[at];
      const int64_t busy = (q.chans + kM - 1) / kM * ((q.rows + sh[1 - at].bn - 1) / sh[1 - at].bn) * sh[1 - at].split;
      const int64_t room = (h->sms - busy) / sh[at].group;
      const int64_t tiles = (mine.chans + sh[at].group * kM - 1) / (sh[at].group * kM) *
                            ((mine.rows + sh[at].bn - 1) / sh[at].bn);
      if (room > 0 && (tiles + room - 1) / room * sh[at].tile < sh[1 - at].clocks) most = static_cast<int>(room);
    }
    if (launch<T, P>(h, p + at, sh + at, 1, sums, early || i, i > 0, most, st)) return -1;
    sums = ColumnSums{};
  }
  return 0;
}

}  // namespace

namespace ptb {

int tc_setup(pt_b200_ops *h) {
  const void *const kernels[] = {
      reinterpret_cast<const void *>(tc_kernel<float, 3>(1, true)),
      reinterpret_cast<const void *>(tc_kernel<float, 3>(2, true)),
      reinterpret_cast<const void *>(tc_kernel<__nv_bfloat16, 1>(1, false)),
      reinterpret_cast<const void *>(tc_kernel<__nv_bfloat16, 1>(2, false)),
      reinterpret_cast<const void *>(tc_kernel<__nv_bfloat16, 1>(1, true)),
      reinterpret_cast<const void *>(tc_kernel<__nv_bfloat16, 1>(2, true)),
      reinterpret_cast<const void *>(tc_kernel<__half, 1>(1, false)),
      reinterpret_cast<const void *>(tc_kernel<__half, 1>(2, false)),
      reinterpret_cast<const void *>(tc_kernel<__half, 1>(1, true)),
      reinterpret_cast<const void *>(tc_kernel<__half, 1>(2, true))};
  for (const void *k : kernels)
    PTB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  for (int log = 0; log < 4; ++log) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(h->sms / (1 << log) << log));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1 << log;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    PTB_CUDA(cudaOccupancyMaxActiveClusters(&h->clusters[log], kernels[log == 1 ? 1 : 0], &cfg));
    PTB_REQUIRE(h->clusters[log] > 0, "pt_b200: no cluster of %d blocks fits this GPU", 1 << log);
  }
  return 0;
}

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

static int prep_lanes(int64_t cols) {
  int lanes = 1;
  while (lanes < 32 && lanes * 8 < cols) lanes *= 2;
  return lanes;
}

int tc_row_blocks(const pt_b200_ops *h, int64_t rows, int64_t cols) {
  const int lanes = prep_lanes(cols), height = kPrepBlock / lanes;
  const int64_t col_blocks = (cols + lanes * 8 - 1) / (lanes * 8);
  const int64_t want = (rows + height * kPrepRows - 1) / (height * kPrepRows);
  const int64_t cap = std::max<int64_t>(1, static_cast<int64_t>(h->sms) * kPrepPerSm / col_blocks);
  return static_cast<int>(std::min(want, cap));
}

void tc_add_job(const pt_b200_ops *h, int dtype, PrepJobs *jobs, int *n, PrepJob a) {
  const int v = 16 / dtype_bytes(dtype);
  a.lanes = prep_lanes(a.cols);
  a.col_blocks = static_cast<int>((a.cols + a.lanes * 8 - 1) / (a.lanes * 8));
  a.row_blocks = tc_row_blocks(h, a.rows, a.cols);
  auto aligned = [&](const void *p, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a.rows == 1 || ld % v == 0);
  };
  a.vec = a.cols % 8 == 0 && aligned(a.src, a.ld) && (!a.act || aligned(a.pre, a.ldp));
  jobs->j[*n] = a;
  const int first = *n ? jobs->end[*n - 1] : 0;
  for (int i = *n; i < kMaxJobs; ++i) jobs->end[i] = first + a.col_blocks * a.row_blocks;
  ++*n;
}

int tc_prep(int dtype, const PrepJobs &jobs, int n, cudaStream_t st) {
  if (n == 0) return 0;
  return with_dtype(dtype, [&](auto *z) -> int {
    prep_kernel<std::remove_pointer_t<decltype(z)>><<<jobs.end[n - 1], kPrepBlock, 0, st>>>(jobs);
    PTB_CUDA(cudaGetLastError());
    count_launch();
    return 0;
  });
}

int tc_products(const pt_b200_ops *h, int dtype, const TcProduct *p, int count, const ColumnSums &sums, bool early,
                cudaStream_t st) {
  switch (dtype) {
    case PT_B200_F32: return launch_products<float, 3>(h, p, count, sums, early, st);
    case PT_B200_BF16: return launch_products<__nv_bfloat16, 1>(h, p, count, sums, early, st);
    default: return launch_products<__half, 1>(h, p, count, sums, early, st);
  }
}

}  // namespace ptb
