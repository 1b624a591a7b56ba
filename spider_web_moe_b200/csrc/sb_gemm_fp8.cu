// Products of block-scaled fp8 matrices on the fp8 tensor cores (tcgen05
// kind::f8f6f4), plain or grouped by expert.
//
//   y[r, c] = sum_kb sa[r, kb] sb[c / 128, kb] sum_{k in kb} a[r, k] b[c, k]
//
// The scales change every 128 elements of k and are arbitrary fp32 numbers, so
// the tensor core can only sum one block of 128 at a time: it writes each
// block's product to one of two TMEM accumulators, and the epilogue warps read
// it back, scale it and add it to sums in their registers, while the tensor
// core fills the other accumulator.
//
// Orientation: token rows are the MMA's M side (one per TMEM lane), weight rows
// its N side (2 x 128 per tile).  An epilogue thread then holds one token row,
// whose scale is one register, and 64 columns of each 128-row weight block,
// whose scale is another: one multiply-add per element, two at a time
// (fma.rn.f32x2).  A SwiGLU tile holds the gate and the up rows of the same 128
// features, so the activation and its quantisation for the next product (a
// 1 x 128 block is the two threads of one token row) need no pass over memory
// of their own.
//
// Three schedules.  One CTA per tile of 128 rows (small groups, quantised outputs);
// CTA pairs for tiles of 256 rows (cta_group::2): each CTA loads its own 128
// rows of a and half of the weight rows, which halves the weight traffic into
// shared memory, the limit of the one-CTA tile; and one with the roles swapped
// for decode batches (second half of this file).
//
// Scales come through shared memory from a warp of their own, which works up to
// four blocks ahead: it loads a block's scales, multiplies them, writes them to
// one of four slots and arrives on the block's barrier (done) beside the MMAs'
// commit, so that the epilogue's one wait finds both.  The epilogue's one arrival
// per block (released) frees the accumulator for the MMAs two blocks on and the
// scale slot for the scale warp four blocks on.
//
// What bounds the pair schedule (16384 x 4096 x 8192, 576 to 594 us on different
// GPUs, about 1300 clocks a block of k where its MMAs take 541).  Measured at 594 us:
// without the additions 448, without the TMEM loads 487, without either 455.  So
// loads and additions account for 300 of the 760 clocks above the MMAs; the other
// 460 are the hand-overs between the roles (commit to wait, release to issue,
// operands arriving), which these times do not split further.  Accumulators in
// halves of 128 columns, each released by itself, took 680 us (every MMA reads its
// rows again); 16-column loads and other orders of loads and additions 580 to 600;
// two plain additions for a packed one 719; the scales' barrier waited for by itself
// 596 (576 as it is).
//
// Warps: 0-7 epilogue (TMEM lane quarter w % 4, columns part w / 4), 8 TMA, 9
// MMA (+TMEM), 10 scales.  Every wait is bounded (sb_common.cuh); loads use no
// multicast.
#include "sb_fp8.cuh"
#include "sb_gemm_common.cuh"
#include "sb_internal.h"

namespace sb {

constexpr int kF8MaxG = 1024;

template <bool kPair>
struct F8Cfg {
  static constexpr int kBM = 128;                      // rows per CTA
  static constexpr int kItemRows = kPair ? 256 : 128;  // rows per item
  static constexpr int kHalf = 128, kBK = 128;
  static constexpr int kABytes = kBM * kBK;
  static constexpr int kHalfBytes = kHalf * kBK;
  static constexpr int kBBytes = kHalfBytes * (kPair ? 1 : 2);  // weight rows this CTA holds
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 4;
  static constexpr int kAccCols = 2 * kHalf;
  static constexpr int kTmemCols = 2 * kAccCols;
  static constexpr int kParts = 2;                     // epilogue warps per TMEM lane quarter
  static constexpr int kCols = kHalf / kParts;         // columns of each half per epilogue thread
  static constexpr int kEpiWarps = 4 * kParts;
  static constexpr int kThreads = (kEpiWarps + 4) * 32;  // whole warpgroups: registers move between them
  // Registers per thread at launch (65536 / kThreads, in steps of 8) and after
  // the split.  The compiler spills in all of these kernels: 34 bytes a thread in the
  // pair's, 90 to 160 in most, 310 with GELU.
  static constexpr int kRegsLaunch = 168, kRegsEpi = 224, kRegsLoad = 56;
  static_assert(kEpiWarps * 32 * kRegsEpi + 128 * kRegsLoad <= kThreads * kRegsLaunch, "the split must fit the launch's registers");
  static constexpr int kSmallRows = 32;                // rows of the box that short tiles load
  static constexpr int kOffA = 0;
  static constexpr int kOffB = kOffA + kStages * kABytes;
  // output staging of the pair schedule: two boxes of 32 rows x 128 bytes per epilogue warp
  static constexpr int kBoxBytes = 32 * 128;
  static constexpr int kOffOut = kOffB + kStages * kBBytes;
  static constexpr int kOffBar = kOffOut + (kPair ? kEpiWarps * 2 * kBoxBytes : 0);
  static constexpr int kOffMisc = kOffBar + (2 * kStages + 4) * 8;
  static constexpr int kOffMax = (kOffMisc + 64 + 15) / 16 * 16;                            // uint32 [2 blocks][kParts][128 rows]
  // What the epilogue needs once per item, from the scale warp: bias of the tile's
  // 256 columns, row scale of its 128 rows.  The scale warp is at most four blocks,
  // so at most four items, ahead of the item whose epilogue runs.
  static constexpr int kItemSlots = 8, kItemFloats = 2 * kHalf + kBM;
  static constexpr int kOffItem = kOffMax + 2 * kParts * kBM * 4;          // float [kItemSlots][kItemFloats]
  static constexpr int kOffScale = kOffItem + kItemSlots * kItemFloats * 4;  // float [4 blocks][kScaleFloats]
  static constexpr int kScaleFloats = kBM + 2 * kHalf;  // [2][128 rows] products, or [128] a and [256] b (kBRows)
  static constexpr int kOffPrefix = kOffScale + 4 * kScaleFloats * 4;      // int [kF8MaxG + 1]
  static constexpr int kOffOffsets = kOffPrefix + (kF8MaxG + 1) * 4;
  static constexpr int kSmemBytes = kOffOffsets + (kF8MaxG + 1) * 4 + 1024;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
  static_assert(kTmemCols == 512, "two accumulators of 256 columns");
  static_assert(kStages == 4, "a block's stage and its scale slot have one number");
  static_assert(kOffItem % 16 == 0 && kOffScale % 16 == 0, "16-byte reads");
};

// Instruction descriptor: e4m3 x e4m3 -> fp32, both K-major, M x N tile.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// Operand descriptors (K-major, 128-byte swizzle; smem_desc_k_sw128) in halves:
// the upper one is constant, the lower one counts 16-byte units, so a stage or a
// step of 32 elements is one addition.  The MMA loop is one thread's chain of
// dependent instructions, and at four short MMAs a round its length shows: with
// descriptors built from addresses, stage numbers from divisions and a barrier of
// its own for the accumulators, a round took 460-500 ns where its MMAs take 260.
constexpr uint32_t kF8DescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
SB_DEVINL uint32_t f8_desc_lo(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }
SB_DEVINL uint64_t f8_desc(uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "n"(kF8DescHi));
  return d;
}
// One lane of a converged warp, which runs the TMA or the MMA loop.  Elected rather
// than `lane == 0`, so that the compiler knows there is one thread: the operands of
// tcgen05.mma and of the TMA copies are uniform registers, and filling them from a
// divergent warp made the four MMAs of a block take 400 clocks to issue (157 so).
SB_DEVINL bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
SB_DEVINL const float* sa_ptr_at(const float* p, int j, int64_t row, int kk, int64_t block) {
  return p + 32 * j * row + kk * block;
}
// A position in a ring of kN slots and the parity of the current round.
template <int kN>
struct Ring {
  int slot = 0;
  uint32_t parity = 0;
  SB_DEVINL void next() {
    if (++slot == kN) {
      slot = 0;
      parity ^= 1;
    }
  }
};

template <bool kPair>
SB_DEVINL void tc_mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 lanes x 32 bit, kN consecutive columns per thread, in pairs of columns.
template <int kN>
SB_DEVINL void tmem_ld_pairs(uint32_t taddr, uint64_t (&v)[kN / 2]) {
  static_assert(kN == 16 || kN == 32, "x16 or x32 loads");
  uint32_t r[kN];
#define SB_R8(i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
  if constexpr (kN == 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : SB_R8(0), SB_R8(8), SB_R8(16), SB_R8(24)
        : "r"(taddr)
        : "memory");
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : SB_R8(0), SB_R8(8)
        : "r"(taddr)
        : "memory");
#undef SB_R8
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) asm("mov.b64 %0, {%1, %2};" : "=l"(v[i]) : "r"(r[2 * i]), "r"(r[2 * i + 1]));
}
// Arrive on a barrier of the pair's leader.  What it hands over is an accumulator and
// nothing else (scales and their slots stay within a CTA and its own barriers),
// ordered by the tcgen05 fences on both sides, so the default CTA-scope release
// does: a cluster-scope one waits for every outstanding access of the thread,
// once per block of k (16384 x 4096 x 8192: 1190 us with it, 685 us without, in a
// form of the kernel that took 685).
SB_DEVINL void mbar_arrive_leader(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Two loads of 32 columns in flight, each in the registers after tmem_wait.
struct Cols32 {
  uint32_t r[32];
};
#define SB_R8(M, r, i) M(r[i]), M(r[i + 1]), M(r[i + 2]), M(r[i + 3]), M(r[i + 4]), M(r[i + 5]), M(r[i + 6]), M(r[i + 7])
SB_DEVINL void tmem_start32(uint32_t taddr, Cols32& c) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : SB_R8("=r", c.r, 0), SB_R8("=r", c.r, 8), SB_R8("=r", c.r, 16), SB_R8("=r", c.r, 24)
      : "r"(taddr)
      : "memory");
}
SB_DEVINL void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps uses of c behind the tmem_wait before it.
SB_DEVINL void tmem_landed(Cols32& c) {
  asm volatile("" : SB_R8("+r", c.r, 0), SB_R8("+r", c.r, 8), SB_R8("+r", c.r, 16), SB_R8("+r", c.r, 24));
}
#undef SB_R8
SB_DEVINL uint64_t pair_at(const Cols32& c, int i) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(c.r[2 * i]), "r"(c.r[2 * i + 1]));
  return v;
}
SB_DEVINL uint64_t pair_of(float x) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
  return r;
}
SB_DEVINL void fma_pair(uint64_t& acc, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}
SB_DEVINL uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// GELU for values that are quantised next: erfc(z) = (a1 t + ... + a5 t^5) exp(-z^2)
// by Abramowitz & Stegun 7.1.26 (erf_as7126's formula), |error| <= 1.5e-7, and
// for x < 0 without a difference, so that the left tail keeps its relative
// precision: 5e-4 of the value at x = -4 and 4e-3 at -6, where the block of a row
// may have nothing larger.  (64 experts x 256 rows x 2048 -> 1024 features: 93 us;
// 7.1.28, without an exponential, 87 us, but off by 4e-3 at -4 and a quarter of the
// value at -6.)  The clamp keeps infinities out of 0 * inf.
SB_DEVINL float gelu_fp8out(float x) {
  const float z = fabsf(x) * 0.70710678118654752f;
  const float t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f));
  const float poly =
      fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t, -0.284496736f), t, 0.254829592f) * t;
  const float c = poly * __expf(-z * z);
  const float h = 0.5f * fminf(fmaxf(x, -1e30f), 1e30f);
  return x > 0.0f ? fmaf(-h, c, x) : h * c;
}

// One item of the schedule: the rows of this CTA of one row tile of one group,
// and a column tile.
struct F8Item {
  int g;
  int row0;    // first row of this CTA
  int rows;    // valid rows of this CTA (may be <= 0 in a pair)
  int peer;    // valid rows of the item's other CTA (pair only)
  int n0;
};
template <bool kPair>
SB_DEVINL F8Item f8_item(const int* prefix, const int* s_off, int G, int n_tiles, int tile_cols, int max_rows, int t,
                         int rank) {
  using C = F8Cfg<kPair>;
  int lo = 0, hi = G - 1;
  while (lo < hi) {  // largest g with prefix[g] <= t
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int local = t - prefix[lo];
  const int mt = local / n_tiles;
  const int tile_row0 = s_off[lo] + mt * C::kItemRows;
  const int left = min(s_off[lo + 1], max_rows) - tile_row0;
  F8Item i;
  i.g = lo;
  i.row0 = tile_row0 + rank * C::kBM;
  i.rows = min(left - rank * C::kBM, C::kBM);
  i.peer = kPair ? min(left - (1 - rank) * C::kBM, C::kBM) : 0;
  i.n0 = (local - mt * n_tiles) * tile_cols;
  return i;
}

SB_DEVINL uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// 16-byte chunk of a row of a staging box (rows of 128 bytes, 128-byte swizzle).
SB_DEVINL uint4* box_chunk(uint8_t* box, int row, int chunk) {
  return reinterpret_cast<uint4*>(box + row * 128 + ((chunk ^ (row & 7)) << 4));
}

// kN consecutive outputs of one row, `valid` of them in range.
template <typename T, int kN>
SB_DEVINL void store_row(T* __restrict__ dst, const float (&v)[kN], int valid, bool vec) {
  if (vec && valid >= kN) {
#pragma unroll
    for (int i = 0; i < kN; i += 16 / sizeof(T)) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      } else {
        *reinterpret_cast<uint4*>(dst + i) = make_uint4(bf16_pair(v[i], v[i + 1]), bf16_pair(v[i + 2], v[i + 3]),
                                                        bf16_pair(v[i + 4], v[i + 5]), bf16_pair(v[i + 6], v[i + 7]));
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kN; ++i)
    if (i < valid) dst[i] = from_f32<T>(v[i]);
}

template <int EPI, bool kBRows, bool kPair>
__global__ void __launch_bounds__(F8Cfg<kPair>::kThreads, 1)
f8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmAs,
               const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmG,
               const __grid_constant__ CUtensorMap tmO, const sb_fp8_matmul_args p, const int tma_out) {
  static_assert(!kPair || EPI == SB_EPI_LINEAR, "quantised outputs run one CTA per tile");
  using C = F8Cfg<kPair>;
  constexpr int S = C::kStages;
  constexpr bool kGate = EPI == SB_EPI_SWIGLU;
  constexpr bool kQuant = EPI != SB_EPI_LINEAR;
  constexpr int kTileCols = kGate ? C::kHalf : 2 * C::kHalf;
  constexpr int kTmaWarp = C::kEpiWarps, kMmaWarp = C::kEpiWarps + 1, kScaleWarp = C::kEpiWarps + 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);  // a pair uses the leader's
  // A block's MMAs are done and its scales (with an item's first block its bias and
  // row scales) are written: the commit and this CTA's scale warp arrive.  The
  // warp's own arrival orders its stores before the epilogue's reads, which a commit,
  // in a pair the other CTA's, would not.  The stage is free, too.  (The MMAs and the
  // scales of the stage's next use wait until every warp has waited for this one.)
  uint64_t* done = full + S;
  // [4], by block: the epilogue has read the accumulator and the scales.  The
  // leader's of a pair counts both CTAs' warps.
  uint64_t* released = done + S;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  int* prefix = reinterpret_cast<int*>(smem + C::kOffPrefix);
  int* s_off = reinterpret_cast<int*>(smem + C::kOffOffsets);

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform for the compiler too
  const int rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = kPair ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int stride = kPair ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  const int G = p.num_groups;
  const int n_tiles = (p.n + kTileCols - 1) / kTileCols;
  const int nk = (p.k + C::kBK - 1) / C::kBK;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], 2);  // the commit, and this CTA's scale warp
    }
    for (int b = 0; b < 4; ++b) mbar_init(&released[b], C::kEpiWarps * (kPair && rank == 0 ? 2 : 1));
    fence_barrier_init();
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmAs);
    tma_prefetch_desc(&tmB);
    if (kGate) tma_prefetch_desc(&tmG);
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) {
    // items per group -> exclusive prefix (warp scan, 32 groups at a time)
    int seen = 0;
    for (int base = 0; base < G; base += 32) {
      const int gi = base + lane;
      int tiles = 0;
      if (gi < G) {
        const int o0 = group_offset(p.offsets, gi, p.max_rows), o1 = group_offset(p.offsets, gi + 1, p.max_rows);
        s_off[gi] = o0;
        if (gi == G - 1) s_off[G] = o1;
        const int lo = min(o0, p.max_rows), hi = min(o1, p.max_rows);
        tiles = hi > lo ? (hi - lo + C::kItemRows - 1) / C::kItemRows * n_tiles : 0;
      }
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += t;
      }
      if (gi < G) prefix[gi] = seen + incl - tiles;
      seen += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) prefix[G] = seen;
  }
  if constexpr (kPair) {
    __syncwarp();
    cluster_sync();  // both CTAs' barriers exist before either signals the other
  } else {
    __syncthreads();
  }
  const int total = prefix[G];
  if (first >= total) return;  // no item for this CTA (or for either of the pair)
  if (warp == kMmaWarp) {
    if constexpr (kPair) {
      tmem_alloc_pair(s_tmem, C::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(s_tmem, C::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp >= C::kEpiWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsLoad));
    if (warp == kTmaWarp) {
    // ---------------------------------------------------------------- TMA
      if (elect_one()) {
        Ring<S> st;
        int issued = 0;
        bool ok = true;
        for (int t = first; t < total && ok; t += stride) {
          const F8Item w = f8_item<kPair>(prefix, s_off, G, n_tiles, kTileCols, p.max_rows, t, rank);
          const bool second = kGate || w.n0 + C::kHalf < p.n;  // the tile's second 128 weight rows exist
          const int brow = static_cast<int>(w.g * p.b_group_rows) + w.n0;
          auto a_bytes = [&](int rows) {  // a CTA without rows loads none: its lanes are never read
            return static_cast<uint32_t>(rows <= 0 ? 0 : (rows <= C::kSmallRows ? C::kSmallRows * C::kBK : C::kABytes));
          };
          const uint32_t tx = kPair ? a_bytes(w.rows) + a_bytes(w.peer) + 2 * C::kHalfBytes
                                    : a_bytes(w.rows) + C::kHalfBytes * (second ? 2 : 1);
          const CUtensorMap* map_a = w.rows <= C::kSmallRows ? &tmAs : &tmA;
          for (int kk = 0; kk < nk; ++kk, st.next()) {
            uint64_t* const bar = &full[st.slot];
            if (!mbar_wait(&done[st.slot], st.parity ^ 1, p.status, SB_DEVERR_MMA_WAIT)) { ok = false; break; }
            if (issued < S) ++issued;
            const int k0 = kk * C::kBK;
            uint8_t* adst = smem + C::kOffA + st.slot * C::kABytes;
            uint8_t* bdst = smem + C::kOffB + st.slot * C::kBBytes;
            if constexpr (kPair) {
              // both CTAs' bytes count on the leader's barrier.  The MMA takes the
              // first half of its N columns from CTA 0, the second from CTA 1.
              if (rank == 0) mbar_expect_tx(bar, tx);
              const uint32_t lead = mapa_shared(smem_u32(bar), 0);
              tma_load_2d_pair(bdst, kGate && rank == 0 ? &tmG : &tmB, lead, k0,
                               kGate || rank == 0 ? brow : brow + (second ? C::kHalf : C::kHalf / 2));
              if (w.rows > 0) tma_load_2d_pair(adst, map_a, lead, k0, w.row0);
            } else {
              mbar_expect_tx(bar, tx);
              tma_load_2d(bdst, kGate ? &tmG : &tmB, bar, k0, brow);
              if (second) tma_load_2d(bdst + C::kHalfBytes, &tmB, bar, k0, kGate ? brow : brow + C::kHalf);
              tma_load_2d(adst, map_a, bar, k0, w.row0);
            }
          }
        }
        // every stage done with: all copies landed and all commit arrivals in
        for (int i = 0; i < issued; ++i, st.next()) {
          const int slot = (st.slot + S - issued) % S;
          if (!mbar_wait(&done[slot], (st.slot >= issued ? st.parity : st.parity ^ 1), p.status, SB_DEVERR_DRAIN)) break;
        }
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------------------- MMA (a pair's leader)
      if (rank == 0 && elect_one()) {
        Ring<S> st;
        Ring<2> acc;
        Ring<4> rel{2, 1};  // of the block two back
        const uint32_t a_lo = f8_desc_lo(smem_u32(smem + C::kOffA)), b_lo = f8_desc_lo(smem_u32(smem + C::kOffB));
        bool ok = true;
        for (int t = first; t < total && ok; t += stride) {
          const F8Item w = f8_item<kPair>(prefix, s_off, G, n_tiles, kTileCols, p.max_rows, t, rank);
          const bool second = kGate || w.n0 + C::kHalf < p.n;
          const uint32_t idesc = idesc_e4m3_f32(C::kItemRows, second ? 2 * C::kHalf : C::kHalf);
          for (int kk = 0; kk < nk; ++kk, st.next(), acc.next(), rel.next()) {
            ok = mbar_wait(&released[rel.slot], rel.parity, p.status, SB_DEVERR_EPI_WAIT) &&
                 mbar_wait(&full[st.slot], st.parity, p.status, SB_DEVERR_TMA_WAIT);
            if (!ok) break;
            tc_fence_after();
            const uint32_t al = a_lo + st.slot * (C::kABytes >> 4), bl = b_lo + st.slot * (C::kBBytes >> 4);
#pragma unroll
            for (int q = 0; q < C::kBK / 32; ++q)
              tc_mma_f8<kPair>(tmem + acc.slot * C::kAccCols, f8_desc(al + 2 * q), f8_desc(bl + 2 * q), idesc, q > 0);
            if constexpr (kPair) tc_commit_pair(&done[st.slot]);
            else tc_commit(&done[st.slot]);
          }
        }
      }
      __syncwarp();
    } else if (warp == kScaleWarp) {
      // ---------------------------------------------------------------- scales
      Ring<4> rel;
      int item = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += stride, item = (item + 1) % C::kItemSlots) {
        const F8Item w = f8_item<kPair>(prefix, s_off, G, n_tiles, kTileCols, p.max_rows, t, rank);
        const bool second = kGate || w.n0 + C::kHalf < p.n;
        const float* sa_ptr = p.a_scale + static_cast<int64_t>(w.row0 + lane) * p.a_scale_row;
        const float* sb0 = (kGate ? p.b_gate_scale : p.b_scale) + w.g * p.b_scale_group;
        const float* sb1 = p.b_scale + w.g * p.b_scale_group;
        if (!kBRows) {
          sb0 += (w.n0 / 128) * p.b_scale_row;
          sb1 += (w.n0 / 128 + (kGate ? 0 : 1)) * p.b_scale_row;
        } else {
          sb1 += static_cast<int64_t>(w.n0 + lane) * p.b_scale_row;
        }
        constexpr int kAhead = kBRows ? 1 : 2, kB = kBRows ? 8 : 2;
        float sa[kAhead][4], sb[kAhead][kB];
        auto load = [&](int kk, int i) {
          if (kk >= nk) return;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sa[i][j] = lane + 32 * j < w.rows ? *sa_ptr_at(sa_ptr, j, p.a_scale_row, kk, p.a_scale_block) : 0.f;
          }
          if (kBRows) {
#pragma unroll
            for (int j = 0; j < kB; ++j)
              sb[i][j] = w.n0 + lane + 32 * j < p.n ? *sa_ptr_at(sb1, j, p.b_scale_row, kk, p.b_scale_block) : 0.f;
          } else {
            sb[i][0] = sb0[kk * p.b_scale_block];
            sb[i][1] = second ? sb1[kk * p.b_scale_block] : 0.f;
          }
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(i, i);
        for (int kk0 = 0; kk0 < nk && ok; kk0 += kAhead) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (kk0 + i >= nk) break;
            if (!__all_sync(0xffffffffu, mbar_wait(&released[rel.slot], rel.parity ^ 1, p.status, SB_DEVERR_EPI_WAIT))) {
              ok = false;
              break;
            }
            if (i == 0 && kk0 == 0) {
              float* d = reinterpret_cast<float*>(smem + C::kOffItem) + item * C::kItemFloats;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float* bias = kGate && j < 4 ? p.bias_gate : p.bias;
                const int c = w.n0 + lane + 32 * (kGate ? j % 4 : j);
                d[lane + 32 * j] = bias && c < p.n ? bias[w.g * p.bias_group + c] : 0.f;
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
                d[2 * C::kHalf + lane + 32 * j] =
                    p.row_scale && lane + 32 * j < w.rows ? p.row_scale[w.row0 + lane + 32 * j] : 1.f;
            }
            float* f = reinterpret_cast<float*>(smem + C::kOffScale) + rel.slot * C::kScaleFloats;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              f[lane + 32 * j] = kBRows ? sa[i][j] : sa[i][j] * sb[i][0];
              if (!kBRows) f[C::kBM + lane + 32 * j] = sa[i][j] * sb[i][1];
            }
            if (kBRows) {
#pragma unroll
              for (int j = 0; j < kB; ++j) f[C::kBM + lane + 32 * j] = sb[i][j];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&done[rel.slot]);  // S == 4: the block's stage
            rel.next();
            load(kk0 + i + kAhead, i);
          }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsEpi));
    constexpr int NC = C::kCols;
    const int quarter = warp & 3, part = warp >> 2;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + part * NC;
    uint32_t* s_max = reinterpret_cast<uint32_t*>(smem + C::kOffMax);
    const uint32_t released_lead = kPair && rank != 0 ? mapa_shared(smem_u32(released), 0) : 0;
    // One counter of blocks for the rings of stages, accumulators and scales, and
    // one of items: beside 192 registers of sums and columns there is little room.
    static_assert(S == 4 && C::kItemSlots == 8, "ring positions are bits of the counters");
    uint32_t it = 0;
    const int items = (total - first + stride - 1) / stride;
    bool ok = true;
    for (int item = 0; item < items && ok; ++item) {
      const int t = first + item * stride;
      bool warp_live, second;
      {
        const F8Item w = f8_item<kPair>(prefix, s_off, G, n_tiles, kTileCols, p.max_rows, t, rank);
        warp_live = quarter * 32 < w.rows;
        second = kGate || w.n0 + C::kHalf < p.n;
      }
      const int r = quarter * 32 + lane;  // row of this CTA's tile
      uint64_t sum[2][NC / 2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NC / 2; ++i) sum[h][i] = 0;
      for (int kk = 0; kk < nk; ++kk, ++it) {
        const uint32_t slot = it & 3;
        if (!__all_sync(0xffffffffu, mbar_wait(&done[slot], (it >> 2) & 1, p.status, SB_DEVERR_EPI_WAIT))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t0 = lane_addr + (it & 1) * C::kAccCols;
        const float* f = reinterpret_cast<const float*>(smem + C::kOffScale) + slot * C::kScaleFloats;
        const uint64_t s0 = pair_of(f[r]), s1 = kBRows ? s0 : pair_of(f[C::kBM + r]);
        // columns 32 j .. of the warp's 2 x 64: two loads in flight, the second
        // pair over the first pair's additions
        auto add = [&](const Cols32& v, int j) {
          const int h = j >> 1, c = (j & 1) * 32;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            if (kBRows) {
              const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(f + C::kBM + h * C::kHalf + part * NC + c + 2 * i);
              fma_pair(sum[h][c / 2 + i], mul_pair(pair_at(v, i), b.x), s0);
              fma_pair(sum[h][c / 2 + i + 1], mul_pair(pair_at(v, i + 1), b.y), s0);
            } else {
              fma_pair(sum[h][c / 2 + i], pair_at(v, i), h ? s1 : s0);
              fma_pair(sum[h][c / 2 + i + 1], pair_at(v, i + 1), h ? s1 : s0);
            }
          }
        };
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&released[slot]);
            if (kPair && rank != 0) mbar_arrive_leader(released_lead + 8u * slot);
          }
        };
        if (warp_live && kBRows) {
          // one load at a time: the scales of the columns need the registers
          Cols32 v;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < 2 || second) {
              tmem_start32(t0 + (j >> 1) * C::kHalf + (j & 1) * 32, v);
              tmem_wait();
              tmem_landed(v);
              add(v, j);
            }
          release();  // only now: add reads the slot's scales
        } else if (warp_live) {
          Cols32 va, vb;
          tmem_start32(t0, va);
          tmem_start32(t0 + 32, vb);
          tmem_wait();
          tmem_landed(va);
          tmem_landed(vb);
          if (second) {
            add(va, 0);
            tmem_start32(t0 + C::kHalf, va);
            add(vb, 1);
            tmem_start32(t0 + C::kHalf + 32, vb);
            tmem_wait();
            tmem_landed(va);
            tmem_landed(vb);
            release();
            add(va, 2);
            add(vb, 3);
          } else {
            add(va, 0);
            add(vb, 1);
            release();
          }
        } else {
          release();
        }
      }
      // the item again, so that its fields need no registers beside the sums
      int t_again = first + item * stride;
      asm volatile("" : "+r"(t_again));
      const F8Item w = f8_item<kPair>(prefix, s_off, G, n_tiles, kTileCols, p.max_rows, t_again, rank);
      const bool live = r < w.rows;
      const int64_t row = w.row0 + r;
      const float* s_bias = reinterpret_cast<const float*>(smem + C::kOffItem) + (item & 7) * C::kItemFloats + part * NC;
      float acc[2][NC];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NC / 2; ++i)
          asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[h][2 * i]), "=f"(acc[h][2 * i + 1]) : "l"(sum[h][i]));
      if constexpr (!kQuant) {
        if (!ok || !warp_live) continue;
        const float rs = s_bias[2 * C::kHalf - part * NC + r];
        // whole boxes of 32 rows leave through shared memory; element stores would keep
        // the warp, and with it the tensor core, waiting for 16-byte pieces of 32
        // different rows.  The hardware clips a box at n, but in units of 16 bytes:
        // where n is no multiple of that (tma_out 1), a box that holds the end is
        // stored by element, or zeros would land behind the row
        const bool staged = kPair && tma_out && quarter * 32 + 32 <= w.rows;
        uint8_t* box = smem + C::kOffOut + warp * 2 * C::kBoxBytes;
        if (staged) {
          if (lane == 0) tma_store_wait_read();  // the previous item's boxes have left
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c0 = w.n0 + h * C::kHalf + part * NC;
          const int valid = p.n - c0;
          if (valid <= 0) continue;
          if (p.bias) {
#pragma unroll
            for (int i = 0; i < NC; i += 4) {
              if (i % 16 == 0) asm volatile("" ::: "memory");  // keeps the loads from piling up in registers
              const float4 b = *reinterpret_cast<const float4*>(s_bias + h * C::kHalf + i);
              acc[h][i] += b.x; acc[h][i + 1] += b.y; acc[h][i + 2] += b.z; acc[h][i + 3] += b.w;
            }
          }
          if (p.row_scale) {
#pragma unroll
            for (int i = 0; i < NC; ++i) acc[h][i] *= rs;
          }
          if (staged && (valid >= NC || tma_out > 1)) {
            if (p.out_dtype == SB_F32) {
              if (h == 1) {
                if (lane == 0) tma_store_wait_read();
                __syncwarp();
              }
#pragma unroll
              for (int i = 0; i < NC; i += 4)
                *box_chunk(box + (i / 32) * C::kBoxBytes, lane, i % 32 / 4) =
                    make_uint4(__float_as_uint(acc[h][i]), __float_as_uint(acc[h][i + 1]),
                               __float_as_uint(acc[h][i + 2]), __float_as_uint(acc[h][i + 3]));
            } else {
#pragma unroll
              for (int i = 0; i < NC; i += 8)
                *box_chunk(box + h * C::kBoxBytes, lane, i / 8) =
                    make_uint4(bf16_pair(acc[h][i], acc[h][i + 1]), bf16_pair(acc[h][i + 2], acc[h][i + 3]),
                               bf16_pair(acc[h][i + 4], acc[h][i + 5]), bf16_pair(acc[h][i + 6], acc[h][i + 7]));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              const int row0 = w.row0 + quarter * 32;
              if (p.out_dtype == SB_F32) {
                tma_store_2d(&tmO, box, c0, row0);
                if (valid > 32) tma_store_2d(&tmO, box + C::kBoxBytes, c0 + 32, row0);
              } else {
                tma_store_2d(&tmO, box + h * C::kBoxBytes, c0, row0);
              }
            }
            continue;
          }
          if (!live) continue;
          if (p.out_dtype == SB_F32) {
            float* dst = static_cast<float*>(p.out) + row * p.ldo + c0;
            store_row(dst, acc[h], valid, reinterpret_cast<uintptr_t>(dst) % 16 == 0);
          } else {
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + c0;
            store_row(dst, acc[h], valid, reinterpret_cast<uintptr_t>(dst) % 16 == 0);
          }
        }
      } else {
        // activation, then one 1 x 128 block per row (SwiGLU) or two (GELU), each
        // held by the threads of the row in the quarter's two warps
        constexpr int kBlocks = kGate ? 1 : 2;
        if (warp_live) {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            const int c0 = w.n0 + b * C::kHalf + part * NC;
            const int valid = p.n - c0;
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < NC; i += 4) {
              if (i % 16 == 0) asm volatile("" ::: "memory");  // keeps the loads from piling up in registers
              const float4 b0 = *reinterpret_cast<const float4*>(s_bias + b * C::kHalf + i);  // SwiGLU: of the gate
              const float bv[4] = {b0.x, b0.y, b0.z, b0.w};
              float uv[4] = {0.f, 0.f, 0.f, 0.f};
              if (kGate) {
                const float4 b1 = *reinterpret_cast<const float4*>(s_bias + C::kHalf + i);
                uv[0] = b1.x; uv[1] = b1.y; uv[2] = b1.z; uv[3] = b1.w;
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float y = acc[b][i + j] + bv[j];
                y = kGate ? silu_bf16out(y) * (acc[1][i + j] + uv[j]) : gelu_fp8out(y);
                y = i + j < valid ? y : 0.f;
                acc[b][i + j] = y;
                m = max(m, abs_bits(y));
              }
            }
            s_max[(b * C::kParts + part) * C::kBM + r] = m;
          }
        }
        ok = named_bar_and(1 + quarter, 32 * C::kParts, ok);
        if (live && ok) {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            const int c0 = w.n0 + b * C::kHalf + part * NC;
            if (w.n0 + b * C::kHalf >= p.n) continue;
            uint32_t m = 0;
#pragma unroll
            for (int q = 0; q < C::kParts; ++q) m = max(m, s_max[(b * C::kParts + q) * C::kBM + r]);
            const Fp8Scale s = fp8_scale(m);
            if (part == 0) p.out_scale[row * p.out_scale_row + (w.n0 / 128 + b) * p.out_scale_block] = s.scale;
            uint8_t* dst = static_cast<uint8_t*>(p.out) + row * p.ldo + c0;
#pragma unroll
            for (int i = 0; i < NC; i += 16) {
              uint32_t q[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                q[k] = fp8_pack4(acc[b][i + 4 * k] * s.inv, acc[b][i + 4 * k + 1] * s.inv,
                                 acc[b][i + 4 * k + 2] * s.inv, acc[b][i + 4 * k + 3] * s.inv);
              if (c0 + i + 16 <= p.n) {
                *reinterpret_cast<uint4*>(dst + i) = make_uint4(q[0], q[1], q[2], q[3]);
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (c0 + i + j < p.n) dst[i + j] = static_cast<uint8_t>(q[j >> 2] >> (8 * (j & 3)));
              }
            }
          }
        }
        named_bar_sync(1 + quarter, 32 * C::kParts);  // s_max is free for the next item
      }
    }
  }
  if (kPair && warp < C::kEpiWarps && lane == 0) tma_store_wait_all();  // stores done before the CTA leaves
  __syncwarp();
  tc_fence_before();
  if constexpr (kPair) cluster_sync();  // neither CTA leaves while the other may still signal it
  else __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair(tmem, C::kTmemCols);
    else tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ------------------------------------------------------------------ few rows
//
// Decode batches: a handful of rows per group, weights streamed once.  The roles
// are swapped: 128 weight rows are the MMA's M side (the TMEM lanes), the kN
// token rows its N side, so scaling and adding a block's kN columns is spread
// over all four lane quarters instead of over the one quarter that a few token
// rows fill (measured on 128 experts x 2048 x 768 at 16 rows each: the up product
// 137 us with rows as M).  A thread holds one output feature and half of the
// token columns; a SwiGLU item has a gate and an up tile, so the thread has both.
// Row tiles of a group are neighbours in the schedule, so their weight tiles
// meet in L2.
//
// LINEAR problems with fewer items than SMs split k over the CTAs of a cluster,
// whose partial sums are added in rank order through distributed shared memory:
// one launch, no workspace, the same result every time.
//
// Warps: 0-7 epilogue (quarter w % 4, columns half w / 4), 8 TMA, 9 MMA (+TMEM),
// 10 scales (as in the kernel above).
template <int EPI, int kN>
struct F8DecCfg {
  static constexpr bool kGate = EPI == SB_EPI_SWIGLU;
  static constexpr int kTiles = kGate ? 2 : 1;  // 128-row weight tiles per item
  static constexpr int kWBytes = 128 * 128;
  static constexpr int kXBytes = kN * 128;
  static constexpr int kStageBytes = kTiles * kWBytes + kXBytes;
  static constexpr int kStagesRaw = (190 * 1024) / kStageBytes;
  static constexpr int kStages = kStagesRaw > 10 ? 10 : kStagesRaw;
  static constexpr int kAcc = 4;  // accumulators in flight between the MMAs and the epilogue
  static constexpr int kAccCols = kTiles * kN;
  static constexpr int kTmemCols = kAcc * kAccCols < 32 ? 32 : kAcc * kAccCols;
  static constexpr int kThreads = 352;
  static constexpr int kCols = kN / 2;  // columns per epilogue thread and tile
  static constexpr int kOffX = kStages * kTiles * kWBytes;
  static constexpr int kOffBar = kOffX + kStages * kXBytes;
  static constexpr int kOffMisc = kOffBar + (2 * kStages + kAcc) * 8;
  static constexpr int kOffScale = (kOffMisc + 16 + 15) / 16 * 16;         // float [kAcc][kTiles][kN]
  static constexpr int kOffMax = kOffScale + kAcc * kTiles * kN * 4;       // uint32 [kN][4 quarters]
  static constexpr int kOffPrefix = kOffMax + kN * 4 * 4;
  static constexpr int kOffOffsets = kOffPrefix + (kF8MaxG + 1) * 4;
  static constexpr int kSmemBytes = kOffOffsets + (kF8MaxG + 1) * 4 + 1024;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
  static_assert(kTmemCols <= 512, "accumulators");
  static_assert(kStages >= kAcc, "a stage's barrier is waited for before its next use completes");
  static_assert(kTiles * kN * 128 * 4 <= kOffX, "the split's partial sums reuse the weight stages");
};

template <int kN>
SB_DEVINL void tmem_ld_cols(uint32_t taddr, uint64_t (&v)[kN / 2]) {
  if constexpr (kN == 8) {
    uint32_t r[8];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("mov.b64 %0, {%1, %2};" : "=l"(v[i]) : "r"(r[2 * i]), "r"(r[2 * i + 1]));
  } else {
    tmem_ld_pairs<kN>(taddr, v);
  }
}
SB_DEVINL float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Item t -> group, first row, valid rows, first feature; row tiles fastest.
template <int kN>
SB_DEVINL F8Item f8_dec_item(const int* prefix, const int* s_off, int G, int n_tiles, int max_rows, int t) {
  int lo = 0, hi = G - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int local = t - prefix[lo];
  const int end = min(s_off[lo + 1], max_rows);
  const int row_tiles = (end - s_off[lo] + kN - 1) / kN;
  const int nt = local / row_tiles;
  F8Item i;
  i.g = lo;
  i.row0 = s_off[lo] + (local - nt * row_tiles) * kN;
  i.rows = min(end - i.row0, kN);
  i.peer = 0;
  i.n0 = nt * 128;
  return i;
}

template <int EPI, int kN>
__global__ void __launch_bounds__(F8DecCfg<EPI, kN>::kThreads, 1)
f8_decode_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                 const __grid_constant__ CUtensorMap tmG, const sb_fp8_matmul_args p, const int splits) {
  using C = F8DecCfg<EPI, kN>;
  constexpr int S = C::kStages, NT = C::kTiles, NC = C::kCols;
  constexpr bool kGate = C::kGate;
  constexpr bool kQuant = EPI != SB_EPI_LINEAR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* done = full + S;  // stage free, accumulator complete (S >= kAcc), scales written: as above
  uint64_t* acc_empty = done + S;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  int* prefix = reinterpret_cast<int*>(smem + C::kOffPrefix);
  int* s_off = reinterpret_cast<int*>(smem + C::kOffOffsets);

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform for the compiler too
  const int rank = static_cast<int>(blockIdx.x) % splits;  // splits == cluster size
  const int first = static_cast<int>(blockIdx.x) / splits, stride = static_cast<int>(gridDim.x) / splits;
  const int G = p.num_groups;
  const int n_tiles = (p.n + 127) / 128;
  const int nk_all = (p.k + 127) / 128;
  const int kb0 = static_cast<int>(static_cast<int64_t>(nk_all) * rank / splits);
  const int nk = static_cast<int>(static_cast<int64_t>(nk_all) * (rank + 1) / splits) - kb0;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 2);  // the copies, and the scale warp
      mbar_init(&done[s], 2);  // the commit, and the scale warp
    }
    for (int b = 0; b < C::kAcc; ++b) mbar_init(&acc_empty[b], 8);
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
    if (kGate) tma_prefetch_desc(&tmG);
  }
  if (warp == 9) {
    tmem_alloc(s_tmem, C::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) {
    int seen = 0;
    for (int base = 0; base < G; base += 32) {
      const int gi = base + lane;
      int tiles = 0;
      if (gi < G) {
        const int o0 = group_offset(p.offsets, gi, p.max_rows), o1 = group_offset(p.offsets, gi + 1, p.max_rows);
        s_off[gi] = o0;
        if (gi == G - 1) s_off[G] = o1;
        const int lo = min(o0, p.max_rows), hi = min(o1, p.max_rows);
        tiles = hi > lo ? (hi - lo + kN - 1) / kN * n_tiles : 0;
      }
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += t;
      }
      if (gi < G) prefix[gi] = seen + incl - tiles;
      seen += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) prefix[G] = seen;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int total = prefix[G];
  bool ok = true;

  if (warp == 8) {
    // ---------------------------------------------------------------- TMA
    if (elect_one()) {
      Ring<S> st;
      int issued = 0;
      for (int t = first; t < total && ok; t += stride) {
        const F8Item w = f8_dec_item<kN>(prefix, s_off, G, n_tiles, p.max_rows, t);
        const int wrow = static_cast<int>(w.g * p.b_group_rows) + w.n0;
        for (int kk = 0; kk < nk; ++kk, st.next()) {
          uint64_t* const bar = &full[st.slot];
          if (!mbar_wait(&done[st.slot], st.parity ^ 1, p.status, SB_DEVERR_MMA_WAIT)) { ok = false; break; }
          if (issued < S) ++issued;
          mbar_expect_tx(bar, C::kStageBytes);
          const int k0 = (kb0 + kk) * 128;
          uint8_t* wdst = smem + st.slot * NT * C::kWBytes;
          if (kGate) tma_load_2d(wdst, &tmG, bar, k0, wrow);
          tma_load_2d(wdst + (NT - 1) * C::kWBytes, &tmW, bar, k0, wrow);
          tma_load_2d(smem + C::kOffX + st.slot * C::kXBytes, &tmX, bar, k0, w.row0);
        }
      }
      for (int i = 0; i < issued; ++i, st.next()) {
        const int slot = (st.slot + S - issued) % S;
        if (!mbar_wait(&done[slot], (st.slot >= issued ? st.parity : st.parity ^ 1), p.status, SB_DEVERR_DRAIN)) break;
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    // ---------------------------------------------------------------- MMA
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_e4m3_f32(128, kN);
      Ring<S> st;
      Ring<C::kAcc> acc;
      const uint32_t w_lo = f8_desc_lo(smem_u32(smem)), x_lo = f8_desc_lo(smem_u32(smem + C::kOffX));
      for (int t = first; t < total && ok; t += stride) {
        for (int kk = 0; kk < nk; ++kk, st.next(), acc.next()) {
          if (!mbar_wait(&full[st.slot], st.parity, p.status, SB_DEVERR_TMA_WAIT)) { ok = false; break; }
          tc_fence_after();
          const uint32_t wl = w_lo + st.slot * (NT * C::kWBytes >> 4), xl = x_lo + st.slot * (C::kXBytes >> 4);
#pragma unroll
          for (int h = 0; h < NT; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              tc_mma_f8<false>(tmem + acc.slot * C::kAccCols + h * kN, f8_desc(wl + h * (C::kWBytes >> 4) + 2 * q),
                               f8_desc(xl + 2 * q), idesc, q > 0);
          tc_commit(&done[st.slot]);
        }
      }
    }
    __syncwarp();
  } else if (warp == 10) {
    // ---------------------------------------------------------------- scales
    Ring<S> st;
    Ring<C::kAcc> acc;
    constexpr int kAhead = 4, kX = (kN + 31) / 32;
    for (int t = first; t < total && ok; t += stride) {
      const F8Item w = f8_dec_item<kN>(prefix, s_off, G, n_tiles, p.max_rows, t);
      const float* sa_ptr = p.a_scale + static_cast<int64_t>(w.row0 + lane) * p.a_scale_row + kb0 * p.a_scale_block;
      const int64_t wofs = w.g * p.b_scale_group + (w.n0 / 128) * p.b_scale_row + kb0 * p.b_scale_block;
      const float* sw_ptr = p.b_scale + wofs;
      const float* sg_ptr = kGate ? p.b_gate_scale + wofs : nullptr;
      float sa[kAhead][kX], sw[kAhead], sg[kAhead];
      auto load = [&](int kk, int i) {
        if (kk >= nk) return;
#pragma unroll
        for (int j = 0; j < kX; ++j)
          sa[i][j] = lane + 32 * j < w.rows ? *sa_ptr_at(sa_ptr, j, p.a_scale_row, kk, p.a_scale_block) : 0.f;
        sw[i] = sw_ptr[kk * p.b_scale_block];
        if (kGate) sg[i] = sg_ptr[kk * p.b_scale_block];
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) load(i, i);
      for (int kk0 = 0; kk0 < nk && ok; kk0 += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (kk0 + i >= nk) break;
          if (!__all_sync(0xffffffffu, mbar_wait(&acc_empty[acc.slot], acc.parity ^ 1, p.status, SB_DEVERR_EPI_WAIT))) {
            ok = false;
            break;
          }
          float* f = reinterpret_cast<float*>(smem + C::kOffScale) + acc.slot * NT * kN;
#pragma unroll
          for (int j = 0; j < kX; ++j)
            if (lane + 32 * j < kN) {
              if (kGate) f[lane + 32 * j] = sa[i][j] * sg[i];
              f[(NT - 1) * kN + lane + 32 * j] = sa[i][j] * sw[i];
            }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&done[st.slot]);
            mbar_arrive(&full[st.slot]);  // passes the free accumulator on to the MMAs
          }
          st.next();
          acc.next();
          load(kk0 + i + kAhead, i);
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * NC;
    const float* s_f = reinterpret_cast<const float*>(smem + C::kOffScale) + half * NC;
    uint32_t* s_max = reinterpret_cast<uint32_t*>(smem + C::kOffMax);
    float* s_red = reinterpret_cast<float*>(smem);  // [kN][128], splits > 1 only
    Ring<S> st;
    Ring<C::kAcc> ring_acc;
    for (int t = first; t < total && ok; t += stride) {
      const F8Item w = f8_dec_item<kN>(prefix, s_off, G, n_tiles, p.max_rows, t);
      const int feat = w.n0 + quarter * 32 + lane;
      const bool fvalid = feat < p.n;
      const bool warp_live = half * NC < w.rows;  // some token column of this warp is valid
      // the item's operands first: their loads pass under the products
      const float bias = p.bias && fvalid ? p.bias[w.g * p.bias_group + feat] : 0.f;
      const float bgate = kGate && p.bias_gate && fvalid ? p.bias_gate[w.g * p.bias_group + feat] : 0.f;
      const float row_scale = !kQuant && p.row_scale && lane < NC && half * NC + lane < w.rows
                                  ? p.row_scale[w.row0 + half * NC + lane] : 1.f;
      uint64_t sum[NT][NC / 2];
#pragma unroll
      for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int i = 0; i < NC / 2; ++i) sum[h][i] = 0;
      for (int kk = 0; kk < nk; ++kk, st.next(), ring_acc.next()) {
        const int buf = ring_acc.slot;
        if (!__all_sync(0xffffffffu, mbar_wait(&done[st.slot], st.parity, p.status, SB_DEVERR_EPI_WAIT))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_live) {
#pragma unroll
          for (int h = 0; h < NT; ++h) {
            uint64_t v[NC / 2];
            tmem_ld_cols<NC>(lane_addr + buf * C::kAccCols + h * kN, v);
#pragma unroll
            for (int i = 0; i < NC / 2; i += 2) {
              const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(s_f + buf * NT * kN + h * kN + 2 * i);
              fma_pair(sum[h][i], v[i], f.x);
              fma_pair(sum[h][i + 1], v[i + 1], f.y);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
      }
      float acc[NT][NC];
#pragma unroll
      for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int i = 0; i < NC / 2; ++i)
          asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[h][2 * i]), "=f"(acc[h][2 * i + 1]) : "l"(sum[h][i]));
      if constexpr (!kQuant) {
        if (splits > 1) {
          // this CTA's partial sums; every CTA of the cluster then finishes kN /
          // splits columns.  One item per cluster, so the ring is done with.
#pragma unroll
          for (int i = 0; i < NC; ++i) s_red[(half * NC + i) * 128 + quarter * 32 + lane] = acc[0][i];
          break;  // finished below, after the cluster's barrier
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          if (half * NC + i >= w.rows) break;
          const int64_t row = w.row0 + half * NC + i;
          const float v = (acc[0][i] + bias) * __shfl_sync(0xffffffffu, row_scale, i);
          if (!fvalid) continue;
          if (p.out_dtype == SB_F32) static_cast<float*>(p.out)[row * p.ldo + feat] = v;
          else static_cast<__nv_bfloat16*>(p.out)[row * p.ldo + feat] = __float2bfloat16_rn(v);
        }
      } else {
        float y[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const float x = acc[NT - 1][i] + bias;
          y[i] = kGate ? silu_bf16out(acc[0][i] + bgate) * x : gelu_fp8out(x);
          if (!fvalid) y[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          if (half * NC + i >= w.rows) break;
          const uint32_t m = __reduce_max_sync(0xffffffffu, abs_bits(y[i]));
          if (lane == 0) s_max[(half * NC + i) * 4 + quarter] = m;
        }
        ok = named_bar_and(1 + half, 128, ok);
        if (ok) {
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const int col = half * NC + i;
            if (col >= w.rows) break;
            const uint4 m = *reinterpret_cast<const uint4*>(s_max + col * 4);
            const Fp8Scale sc = fp8_scale(max(max(m.x, m.y), max(m.z, m.w)));
            const int64_t row = w.row0 + col;
            if (quarter == 0 && lane == 0) p.out_scale[row * p.out_scale_row + (w.n0 / 128) * p.out_scale_block] = sc.scale;
            if (fvalid)
              static_cast<uint8_t*>(p.out)[row * p.ldo + feat] =
                  static_cast<uint8_t>(fp8_pack4(y[i] * sc.inv, 0.f, 0.f, 0.f));
          }
        }
        named_bar_sync(1 + half, 128);  // s_max is free for the next item
      }
    }
  }
  __syncwarp();
  if (!kQuant && splits > 1) {
    // every CTA of the cluster has its partial sums in place (each has an item:
    // the grid is items x splits for plain products, whose item count the host knows)
    cluster_sync();
    if (warp < 8 && first < total) {
      const F8Item w = f8_dec_item<kN>(prefix, s_off, G, n_tiles, p.max_rows, first);
      const int quarter = warp & 3, half = warp >> 2;
      const int feat = w.n0 + quarter * 32 + lane;
      const float bias = p.bias && feat < p.n ? p.bias[w.g * p.bias_group + feat] : 0.f;
      // columns rank, rank + splits, ...: alternately for the two halves' warps
      for (int col = rank + half * splits; col < w.rows; col += 2 * splits) {
        const uint32_t mine = smem_u32(smem) + (col * 128 + quarter * 32 + lane) * 4;
        float v = 0.f;
        for (int q = 0; q < splits; ++q) v += ld_cluster_f32(mapa_shared(mine, q));
        const int64_t row = w.row0 + col;
        v += bias;
        if (p.row_scale) v *= p.row_scale[row];
        if (feat < p.n) {
          if (p.out_dtype == SB_F32) static_cast<float*>(p.out)[row * p.ldo + feat] = v;
          else static_cast<__nv_bfloat16*>(p.out)[row * p.ldo + feat] = __float2bfloat16_rn(v);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

static bool f8_map(CUtensorMap* m, const void* base, int64_t k, int64_t rows, int64_t pitch, int box_rows) {
  return make_map(m, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, k, rows, pitch, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int EPI, bool kBRows, bool kPair>
static int launch_f8(const sb_fp8_matmul_args& a, cudaStream_t st) {
  using C = F8Cfg<kPair>;
  auto kern = f8_gemm_kernel<EPI, kBRows, kPair>;
  static int configured_device = -1;
  static int max_ctas = 0;  // CTAs (or pairs) that run at once
  int dev = 0;
  cudaGetDevice(&dev);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  if (configured_device != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return cuda_status(e);
    int n = current_sm_count();
    if (kPair) {
      cfg.gridDim = dim3(2 * n);
      cfg.attrs = attr + 1;
      cfg.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess || clusters <= 0) {
        cudaGetLastError();
        clusters = n / 2;
      }
      n = clusters;
    }
    max_ctas = n;
    configured_device = dev;
  }
  constexpr int kTileCols = EPI == SB_EPI_SWIGLU ? C::kHalf : 2 * C::kHalf;
  const int64_t b_rows = (a.num_groups - 1) * a.b_group_rows + a.n;
  CUtensorMap ma, mas, mb, mg;
  if (!f8_map(&ma, a.a, a.k, a.max_rows, a.lda, C::kBM) || !f8_map(&mas, a.a, a.k, a.max_rows, a.lda, C::kSmallRows) ||
      !f8_map(&mb, a.b, a.k, b_rows, a.ldb, C::kHalf))
    return SB_ERR_UNSUPPORTED;
  mg = mb;
  if (EPI == SB_EPI_SWIGLU && !f8_map(&mg, a.b_gate, a.k, b_rows, a.ldb, C::kHalf)) return SB_ERR_UNSUPPORTED;
  // LINEAR outputs of the pair schedule as a tensor of boxes of 32 rows x 128
  // bytes; without one (an unaligned output) every element is stored by its thread
  CUtensorMap mo = ma;
  const int esize = a.out_dtype == SB_F32 ? 4 : 2;
  const bool boxes =
      kPair && EPI == SB_EPI_LINEAR && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.ldo * esize % 16 == 0 &&
      make_map(&mo, a.out, esize == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.n,
               a.max_rows, a.ldo * esize, 128 / esize, 32, CU_TENSOR_MAP_SWIZZLE_128B);
  const int tma_out = boxes ? (static_cast<int64_t>(a.n) * esize % 16 == 0 ? 2 : 1) : 0;  // 2: the end of a row, too
  const int64_t n_tiles = (a.n + kTileCols - 1) / kTileCols;
  const int64_t row_tiles = (a.max_rows + C::kItemRows - 1) / C::kItemRows + (a.offsets ? a.num_groups : 0);
  if (n_tiles * row_tiles > 0x7fffffff) return SB_ERR_UNSUPPORTED;
  const int ctas = static_cast<int>(n_tiles * row_tiles < max_ctas ? n_tiles * row_tiles : max_ctas);
  cfg.gridDim = dim3(kPair ? 2 * ctas : ctas);
  cfg.attrs = pdl_enabled() ? attr : attr + 1;
  cfg.numAttrs = (pdl_enabled() ? 1 : 0) + (kPair ? 1 : 0);
  note_launch();
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, ma, mas, mb, mg, mo, a, tma_out));
}

template <int EPI, int kN>
static int launch_f8_decode(const sb_fp8_matmul_args& a, cudaStream_t st) {
  using C = F8DecCfg<EPI, kN>;
  auto kern = f8_decode_kernel<EPI, kN>;
  static int configured_device = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_device != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return cuda_status(e);
    configured_device = dev;
  }
  const int64_t b_rows = (a.num_groups - 1) * a.b_group_rows + a.n;
  CUtensorMap mx, mw, mg;
  if (!f8_map(&mx, a.a, a.k, a.max_rows, a.lda, kN) || !f8_map(&mw, a.b, a.k, b_rows, a.ldb, 128))
    return SB_ERR_UNSUPPORTED;
  mg = mw;
  if (EPI == SB_EPI_SWIGLU && !f8_map(&mg, a.b_gate, a.k, b_rows, a.ldb, 128)) return SB_ERR_UNSUPPORTED;
  const int64_t n_tiles = (a.n + 127) / 128;
  const int64_t row_tiles = (a.max_rows + kN - 1) / kN + (a.offsets ? (a.num_groups < a.max_rows ? a.num_groups : a.max_rows) : 0);
  const int64_t items = n_tiles * row_tiles;
  if (items > 0x7fffffff) return SB_ERR_UNSUPPORTED;
  const int sms = current_sm_count();
  // k split over clusters of 2, 4 or 8 CTAs while they all fit the GPU at once,
  // with at least two blocks of k each
  int splits = 1;
  if (EPI == SB_EPI_LINEAR && !a.offsets)
    while (splits < 8 && items * splits * 2 <= sms && (a.k + 127) / 128 >= 4 * splits) splits *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits > 1 ? static_cast<int>(items) * splits : static_cast<int>(items < sms ? items : sms));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cfg.attrs = pdl_enabled() ? attr : attr + 1;
  cfg.numAttrs = (pdl_enabled() ? 1 : 0) + (splits > 1 ? 1 : 0);
  note_launch();
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, mx, mw, mg, a, splits));
}

// Column count of the weights-as-M schedule, or 0 for the row-tile schedules.
// Plain products: up to 64 rows it is bound by the weights' bytes.  Beyond, while
// its items of 128 x 64 fit the GPU at once: a block of k takes it about 0.45 us
// and a 256 x 256 pair tile 0.65 us, and the same outputs are eight times the
// items, which can then split k as well (128 x 2048 x 4096: 17.5 us in row tiles,
// 11.8 us so).
//
// Grouped products: by the average rows of a group, all that the host knows.  Times
// with 16 / 32 / 64 columns / row tiles in us, 128 experts with up to two or three
// times the average rows, SwiGLU 2048 -> 2 x 768 and LINEAR 768 -> 2048:
//   rows  4:   68  68  73 101    41  42  46  66
//   rows  8:   77  73  78 104    45  45  50  67
//   rows 24:   98  87  99 105    78  60  66  72
//   rows 32:  115  93 108 105    96  71  71  74
//   rows 40:  136 103 110 106   112  84  76  78
//   rows 48:  152 122 126 109   131  96  86  80  (equal groups: 140 123 116 109, 116 97 74 77)
// GELU as SwiGLU, sooner in row tiles (rows 40: 61 / 67 / 56).  An average does not
// see skew: 256 rows in each of 8 experts and none in 120 take 36 us in 32 columns
// where row tiles take 23.
static int decode_columns(const sb_fp8_matmul_args& a) {
  if (a.b_block_rows != 128) return 0;
  if (!a.offsets) {
    if (a.max_rows <= 32) return a.max_rows <= 16 ? 16 : 32;
    const int64_t items = static_cast<int64_t>((a.max_rows + 63) / 64) * ((a.n + 127) / 128);
    return a.max_rows <= 64 || items <= current_sm_count() ? 64 : 0;
  }
  const int per_group = a.max_rows / a.num_groups;
  return per_group <= 4 ? 16 : (per_group <= 32 ? 32 : (per_group <= 48 && a.epilogue == SB_EPI_LINEAR ? 64 : 0));
}

// LINEAR products: pairs pay when the rows per group fill their 256-row tiles (the
// down product of 64 experts x 256 rows, k 1024, n 2048: 72 us against 100; of
// groups of 0 to 1900 rows 112 against 121).  A quantised epilogue is the tail of
// each item and takes as long in both schedules, so there the halved weight traffic
// buys nothing (up product, k 2048, 2 x 1024: 120 us both; 16 x 1024 rows, k 4096: 370
// against 378) and the half-empty last tiles of the groups cost (uneven groups: 184
// against 149): those products run one CTA per tile.
static bool use_pair(const sb_fp8_matmul_args& a) { return a.max_rows / a.num_groups > 128; }

}  // namespace sb

using namespace sb;

extern "C" SB_API int sb_fp8_matmul(const sb_fp8_matmul_args* args, void* stream) {
  if (!args) return SB_ERR_ARG;
  const sb_fp8_matmul_args& a = *args;
  const bool quant = a.epilogue == SB_EPI_GELU || a.epilogue == SB_EPI_SWIGLU;
  if ((!quant && a.epilogue != SB_EPI_LINEAR) || (!quant && a.out_dtype != SB_F32 && a.out_dtype != SB_BF16) ||
      a.num_groups < 1 || a.num_groups > kF8MaxG || (!a.offsets && a.num_groups != 1) || a.max_rows < 0 ||
      a.max_rows > kMaxExtent || a.n < 1 || a.n > kMaxExtent || a.k < 1 || a.k > kMaxExtent ||
      (a.b_block_rows != 128 && a.b_block_rows != 1) || (quant && a.b_block_rows != 128) ||
      a.lda < a.k || a.lda % 16 || a.ldb < a.k || a.ldb % 16 || (a.num_groups > 1 && a.b_group_rows < a.n) ||
      a.ldo < a.n || (quant && a.ldo % 16))
    return SB_ERR_ARG;
  if (a.max_rows == 0) return SB_OK;
  auto aligned = [](const void* p) { return p && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!aligned(a.a) || !aligned(a.b) || !a.a_scale || !a.b_scale || !a.out || (quant && (!aligned(a.out) || !a.out_scale)) ||
      (a.epilogue == SB_EPI_SWIGLU && (!aligned(a.b_gate) || !a.b_gate_scale)))
    return SB_ERR_ARG;
  if ((a.num_groups - 1) * a.b_group_rows + a.n > 0x7fffffff) return SB_ERR_UNSUPPORTED;  // TMA row coordinates
  if (current_cc_major() != 10) return SB_ERR_NO_DEVICE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SB_F8_DECODE(EPI)                                         \
  do {                                                            \
    if (cols == 16) return launch_f8_decode<EPI, 16>(a, st);      \
    if (cols == 32) return launch_f8_decode<EPI, 32>(a, st);      \
    return launch_f8_decode<EPI, 64>(a, st);                      \
  } while (0)
  if (const int cols = decode_columns(a)) {
    if (a.epilogue == SB_EPI_SWIGLU) SB_F8_DECODE(SB_EPI_SWIGLU);
    if (a.epilogue == SB_EPI_GELU) SB_F8_DECODE(SB_EPI_GELU);
    SB_F8_DECODE(SB_EPI_LINEAR);
  }
#undef SB_F8_DECODE
  if (a.epilogue == SB_EPI_SWIGLU) return launch_f8<SB_EPI_SWIGLU, false, false>(a, st);
  if (a.epilogue == SB_EPI_GELU) return launch_f8<SB_EPI_GELU, false, false>(a, st);
  const bool pair = use_pair(a);
#define SB_F8(ROWS) return pair ? launch_f8<SB_EPI_LINEAR, ROWS, true>(a, st) : launch_f8<SB_EPI_LINEAR, ROWS, false>(a, st)
  if (a.b_block_rows == 1) SB_F8(true);
  SB_F8(false);
#undef SB_F8
}

// ------------------------------------------------------------------ linear layer
namespace sb {

// A quantised matrix in the workspace: rows x cols with 1 x 128 or 128 x 128 blocks.
struct F8Buf {
  uint8_t* q;
  float* s;
  int64_t ld, s_row, s_col;
};
static F8Buf f8_buf(Carver& c, int rows, int cols, int block_rows) {
  F8Buf b;
  const int64_t cb = (cols + 127) / 128;
  b.ld = align_up(cols, 16);
  b.q = c.take<uint8_t>(static_cast<size_t>(rows) * b.ld);
  if (block_rows == 1) {
    b.s_row = 1;
    b.s_col = align_up(rows, 4);
    b.s = c.take<float>(b.s_col * cb);
  } else {
    b.s_row = cb;
    b.s_col = 1;
    b.s = c.take<float>(static_cast<size_t>((rows + 127) / 128) * cb);
  }
  return b;
}
static sb_fp8_quantize_args f8_quantize_args(const F8Buf& b, const void* x, int dtype, int rows, int cols, int64_t x_row,
                                             int64_t x_col, int block_rows) {
  sb_fp8_quantize_args q = {};
  q.x = x; q.dtype = dtype; q.block_rows = block_rows; q.batch = 1; q.rows = rows; q.cols = cols;
  q.x_row = x_row; q.x_col = x_col; q.q = b.q; q.ldq = b.ld;
  q.scale = b.s; q.scale_row = b.s_row; q.scale_col = b.s_col;
  return q;
}
static int f8_quantize(const F8Buf& b, const void* x, int dtype, int rows, int cols, int64_t x_row, int64_t x_col,
                       int block_rows, void* stream) {
  const sb_fp8_quantize_args q = f8_quantize_args(b, x, dtype, rows, cols, x_row, x_col, block_rows);
  return sb_fp8_quantize_blocks(&q, stream);
}
static int f8_product(const F8Buf& a, const F8Buf& b, int b_block_rows, int m, int n, int k, void* out, int out_dtype,
                      int* status, void* stream) {
  sb_fp8_matmul_args g = {};
  g.epilogue = SB_EPI_LINEAR; g.out_dtype = out_dtype; g.num_groups = 1; g.max_rows = m; g.n = n; g.k = k;
  g.a = a.q; g.lda = a.ld; g.a_scale = a.s; g.a_scale_row = a.s_row; g.a_scale_block = a.s_col;
  g.b = b.q; g.ldb = b.ld; g.b_scale = b.s; g.b_scale_row = b.s_row; g.b_scale_block = b.s_col;
  g.b_block_rows = b_block_rows; g.out = out; g.ldo = n; g.status = status;
  return sb_fp8_matmul(&g, stream);
}
static bool f8_sizes_ok(int m, int n, int k) {
  return m >= 0 && m <= kMaxExtent && n >= 1 && n <= kMaxExtent && k >= 1 && k <= kMaxExtent;
}
static bool f8_linear_ok(int dtype, int64_t ldx, int m, int n, int k, int w_dtype) {
  return (dtype == SB_F32 || dtype == SB_BF16) && (w_dtype == SB_F32 || w_dtype == SB_BF16) && f8_sizes_ok(m, n, k) &&
         ldx >= k;
}

}  // namespace sb

extern "C" SB_API size_t sb_fp8_linear_workspace_bytes(int m, int n, int k, int packed) {
  if (!f8_sizes_ok(m, n, k)) return 0;
  Carver c(nullptr, ~size_t(0) >> 1);
  f8_buf(c, m, k, 1);
  if (!packed) f8_buf(c, n, k, 128);
  return align_up(c.used, 256) + 256;
}

extern "C" SB_API int sb_fp8_linear(const void* x, int dtype, int64_t ldx, int m, int n, int k, const void* w,
                                    int w_dtype, int64_t ldw, const float* w_scale, int64_t w_scale_row,
                                    int64_t w_scale_col, void* y, int* status, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (!f8_linear_ok(dtype, ldx, m, n, k, w_dtype) || ldw < k || !w) return SB_ERR_ARG;
  if (m == 0) return SB_OK;
  if (!x || !y) return SB_ERR_ARG;
  Carver c(workspace, workspace_bytes);
  const F8Buf xq = f8_buf(c, m, k, 1);
  F8Buf wq;
  if (w_scale) {
    wq = {const_cast<uint8_t*>(static_cast<const uint8_t*>(w)), const_cast<float*>(w_scale), ldw, w_scale_row,
          w_scale_col};
  } else {
    wq = f8_buf(c, n, k, 128);
  }
  if (!workspace || c.overflow) return SB_ERR_WORKSPACE;
  if (!w_scale) {
    const int rc = f8_quantize(wq, w, w_dtype, n, k, ldw, 1, 128, stream);
    if (rc) return rc;
  }
  const int rc = f8_quantize(xq, x, dtype, m, k, ldx, 1, 1, stream);
  return rc ? rc : f8_product(xq, wq, 128, m, n, k, y, dtype, status, stream);
}

extern "C" SB_API size_t sb_fp8_linear_backward_workspace_bytes(int m, int n, int k) {
  if (!f8_sizes_ok(m, n, k)) return 0;
  Carver c(nullptr, ~size_t(0) >> 1);
  f8_buf(c, m, n, 1);
  f8_buf(c, k, n, 128);
  f8_buf(c, n, m, 1);
  f8_buf(c, k, m, 1);
  return align_up(c.used, 256) + 256;
}

extern "C" SB_API int sb_fp8_linear_backward(const void* x, int dtype, int64_t ldx, int m, int n, int k, const void* w,
                                             int w_dtype, int64_t ldw, const void* dy, int64_t dy_row, int64_t dy_col,
                                             void* dx, void* dw, int* status, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  if (!f8_linear_ok(dtype, ldx, m, n, k, w_dtype) || ldw < k || dy_row < 0 || dy_col < 0) return SB_ERR_ARG;
  if (m == 0) {  // no rows: dw is a sum of none
    if (!dw) return SB_OK;
    return cuda_status(cudaMemsetAsync(dw, 0, static_cast<size_t>(n) * k * (w_dtype == SB_F32 ? 4 : 2),
                                       static_cast<cudaStream_t>(stream)));
  }
  if (!dy || (dx && !w) || (dw && !x)) return SB_ERR_ARG;
  Carver c(workspace, workspace_bytes);
  const F8Buf dq = f8_buf(c, m, n, 1), wt = f8_buf(c, k, n, 128), dt = f8_buf(c, n, m, 1), xt = f8_buf(c, k, m, 1);
  if (!workspace || c.overflow) return SB_ERR_WORKSPACE;
#define SB_TRY(e) do { const int rc = (e); if (rc) return rc; } while (0)
  // dy along its rows for dx and along its columns for dw, in one pass where it can
  const bool both = dx && dw &&
                    fp8_quantize_both(f8_quantize_args(dq, dy, dtype, m, n, dy_row, dy_col, 1),
                                      f8_quantize_args(dt, dy, dtype, n, m, dy_col, dy_row, 1),
                                      static_cast<cudaStream_t>(stream)) == SB_OK;
  if (dx) {  // the blocks of w^T are the transposed blocks of w: the forward pass's values
    SB_TRY(f8_quantize(wt, w, w_dtype, k, n, 1, ldw, 128, stream));
    if (!both) SB_TRY(f8_quantize(dq, dy, dtype, m, n, dy_row, dy_col, 1, stream));
    SB_TRY(f8_product(dq, wt, 128, m, k, n, dx, dtype, status, stream));
  }
  if (dw) {
    if (!both) SB_TRY(f8_quantize(dt, dy, dtype, n, m, dy_col, dy_row, 1, stream));
    SB_TRY(f8_quantize(xt, x, dtype, k, m, 1, ldx, 1, stream));
    SB_TRY(f8_product(dt, xt, 1, n, k, m, dw, w_dtype, status, stream));
  }
#undef SB_TRY
  return SB_OK;
}

// ------------------------------------------------------------------ expert delta
namespace sb {

struct F8DeltaBuffers {
  int32_t *off, *row, *slot, *inv;
  float* w;
  void* group_ws;
  size_t group_ws_bytes;
  uint8_t *xq, *act;
  float *xs, *as, *y;
  int* status;
};

constexpr int kF8MaxExperts = 256;  // as many as sb_group takes

static bool f8_experts_ok(const sb_fp8_experts* x) {
  return x && x->num_experts >= 1 && x->num_experts <= kF8MaxExperts && x->hidden >= 1 && x->hidden <= kMaxExtent &&
         x->ffn >= 1 && x->ffn <= kMaxExtent &&
         (x->activation == SB_ACT_GELU || x->activation == SB_ACT_SWIGLU) && x->ld_in % 16 == 0 && x->ld_in >= x->hidden &&
         x->ld_ffn % 16 == 0 && x->ld_ffn >= x->ffn;
}

// Carves the scratch of one call; returns the bytes it takes.
static size_t f8_carve(const sb_fp8_experts& x, int n, int k, void* ws, size_t bytes, F8DeltaBuffers* b) {
  Carver c(ws, bytes);
  const size_t pairs = static_cast<size_t>(n) * k, pr = align_up(pairs, 4);
  b->status = c.take<int>(kStatusBytes / sizeof(int));
  b->off = c.take<int32_t>(x.num_experts + 1);
  b->row = c.take<int32_t>(pairs);
  b->slot = c.take<int32_t>(pairs);
  b->inv = c.take<int32_t>(pairs);
  b->w = c.take<float>(pairs);
  b->group_ws_bytes = sb_group_workspace_bytes(n, k, x.num_experts);
  b->group_ws = c.take<uint8_t>(b->group_ws_bytes);
  b->xq = c.take<uint8_t>(pairs * align_up(x.hidden, 16));
  b->xs = c.take<float>(pr * ((x.hidden + 127) / 128));
  b->act = c.take<uint8_t>(pairs * align_up(x.ffn, 16));
  b->as = c.take<float>(pr * ((x.ffn + 127) / 128));
  b->y = c.take<float>(pairs * align_up(x.hidden, 4));
  return c.overflow ? static_cast<size_t>(-1) : align_up(c.used, 256);
}

}  // namespace sb

extern "C" SB_API size_t sb_fp8_expert_delta_workspace_bytes(const sb_fp8_experts* experts, int n_tokens, int top_k) {
  if (!f8_experts_ok(experts) || n_tokens < 0 || top_k < 1 || top_k > 64 ||
      static_cast<int64_t>(n_tokens) * top_k > kMaxExtent)
    return 0;
  F8DeltaBuffers b;
  return f8_carve(*experts, n_tokens > 0 ? n_tokens : 1, top_k, nullptr, ~size_t(0) >> 1, &b);
}

extern "C" SB_API int sb_fp8_expert_delta(const sb_fp8_experts* experts, const void* messages, int dtype, int64_t ld,
                                          const int32_t* top_idx, const float* top_w, int n_tokens, int top_k,
                                          void* delta, int delta_dtype, int* status, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  if (!f8_experts_ok(experts) || (dtype != SB_F32 && dtype != SB_BF16) ||
      (delta_dtype != SB_F32 && delta_dtype != SB_BF16) || n_tokens < 0 || top_k < 1 || top_k > 64 ||
      static_cast<int64_t>(n_tokens) * top_k > kMaxExtent || ld < experts->hidden)
    return SB_ERR_ARG;
  if (n_tokens == 0) return SB_OK;
  const sb_fp8_experts& x = *experts;
  const bool swiglu = x.activation == SB_ACT_SWIGLU;
  if (!messages || !top_idx || !top_w || !delta || !x.w_up || !x.s_up || !x.w_down || !x.s_down ||
      (swiglu && (!x.w_gate || !x.s_gate)))
    return SB_ERR_ARG;
  F8DeltaBuffers b;
  const size_t need = f8_carve(x, n_tokens, top_k, workspace, workspace_bytes, &b);
  if (!workspace || need == static_cast<size_t>(-1) || need > workspace_bytes) return SB_ERR_WORKSPACE;
  const int N = n_tokens, E = x.num_experts, H = x.hidden, U = x.ffn, P = N * top_k;
  const int64_t pr = align_up(P, 4);
  const int hb = (H + 127) / 128, ub = (U + 127) / 128;
  if (!status) status = b.status;
#define SB_TRY(e) do { const int rc = (e); if (rc) return rc; } while (0)
  // NaN weights stay (the routing ranks a NaN logit first so that it is seen): they
  // reach the token's delta as the down product's row scale
  SB_TRY(sb_group(top_idx, top_w, N, top_k, E, SB_GROUP_POSITIVE_ONLY | SB_GROUP_KEEP_NAN, b.off, b.row, b.slot, b.w,
                  b.inv, b.group_ws, b.group_ws_bytes, stream));
  sb_fp8_quantize_args q = {};
  q.x = messages; q.dtype = dtype; q.block_rows = 1; q.batch = 1; q.rows = P; q.cols = H;
  q.x_row = ld; q.x_col = 1; q.row_index = b.row; q.row_count = b.off + E;
  q.q = b.xq; q.ldq = align_up(H, 16); q.scale = b.xs; q.scale_row = 1; q.scale_col = pr;
  SB_TRY(sb_fp8_quantize_blocks(&q, stream));
  sb_fp8_matmul_args a = {};
  a.epilogue = swiglu ? SB_EPI_SWIGLU : SB_EPI_GELU;
  a.num_groups = E; a.max_rows = P; a.n = U; a.k = H; a.offsets = b.off; a.status = status; a.b_block_rows = 128;
  a.a = b.xq; a.lda = q.ldq; a.a_scale = b.xs; a.a_scale_row = 1; a.a_scale_block = pr;
  a.b = x.w_up; a.b_gate = x.w_gate; a.ldb = x.ld_in; a.b_group_rows = U;
  a.b_scale = x.s_up; a.b_gate_scale = x.s_gate;
  a.b_scale_row = hb; a.b_scale_block = 1; a.b_scale_group = static_cast<int64_t>(ub) * hb;
  a.bias = x.b_up; a.bias_gate = x.b_gate; a.bias_group = U;
  a.out = b.act; a.ldo = align_up(U, 16); a.out_scale = b.as; a.out_scale_row = 1; a.out_scale_block = pr;
  SB_TRY(sb_fp8_matmul(&a, stream));
  sb_fp8_matmul_args d = {};
  d.epilogue = SB_EPI_LINEAR; d.out_dtype = SB_F32;
  d.num_groups = E; d.max_rows = P; d.n = H; d.k = U; d.offsets = b.off; d.status = status; d.b_block_rows = 128;
  d.a = b.act; d.lda = a.ldo; d.a_scale = b.as; d.a_scale_row = 1; d.a_scale_block = pr;
  d.b = x.w_down; d.ldb = x.ld_ffn; d.b_group_rows = H;
  d.b_scale = x.s_down; d.b_scale_row = ub; d.b_scale_block = 1; d.b_scale_group = static_cast<int64_t>(hb) * ub;
  d.bias = x.b_down; d.bias_group = H; d.row_scale = b.w;
  d.out = b.y; d.ldo = align_up(H, 4);
  SB_TRY(sb_fp8_matmul(&d, stream));
  const int cols = static_cast<int>(align_up(H, 4));
  SB_TRY(sb_combine_rows(b.y, cols, 1, 0, b.inv, top_k, N, cols,
                         delta_dtype == SB_F32 ? static_cast<float*>(delta) : nullptr, nullptr, 0,
                         delta_dtype == SB_F32 ? nullptr : delta, SB_BF16, stream));
#undef SB_TRY
  return SB_OK;
}
