// Gated feed-forward block: forward and backward on the sm_100a tensor cores.
//
//   g = x Wg^T   u = x Wu^T   h = act(g) * u   y = h Wd^T
//   x [T, d], Wg and Wu [f, d], Wd [d, f], 16-bit (BF16 or FP16), FP32 accumulation
//   act(g) = g sigma(z): z = g (SiLU) or z = 2 sqrt(2/pi) (g + 0.044715 g^3) (GELU,
//   tanh form: 0.5 (1 + tanh w) = sigma(2 w))
// and, from x (or its 8-bit checkpoint, restored exactly into 16 bits first):
//   dh = dy Wd          g, u recomputed, s = sigma(z)
//   dg = dh u (s + g s (1 - s) z')      du = dh act(g)      h again for dWd
//   dx = dg Wg + du Wu   dWg = dg^T x   dWu = du^T x   dWd = dy^T h
// h, dg and du are rounded once to 16 bits because they are the next product's
// tensor-core operand; dh is only read by the elementwise step, so it stays FP32
// (rounding it too cost 0.0029 against 0.0023 relative error of the BF16 gradients).
//
// Two kernels do every product:
//
// k_ffn_pair (more tokens, and all weight gradients): the CTA-pair tcgen05
// form of mb_gemm.cu's header (256 x 256 output tile over two SMs, M = 256,
// TMA-fed ring, two TMEM accumulators so that a tile's epilogue overlaps the next
// tile's MMAs), with
//   * operands read in the layout they have: K-major, or MN-major where the
//     contraction runs over rows (dh, dx, dW), so that nothing is transposed;
//   * gate and up as the two halves of one tile's B operand: the even CTA loads 128
//     gate rows, the odd one the same 128 up rows, so a lane's TMEM row holds g in
//     columns 0-127 and u of the same features in 128-255, and h (or dg, du, h from
//     dh, which each lane fetches for its row while the MMAs run) is formed where they
//     lie;
//   * dx as one contraction over both (dg, Wg) and (du, Wu): one accumulator;
//   * dx and the three weight gradients as one launch, dealt so that the pairs end
//     together (mb_ffn_deal.cuh);
//   * long contractions in double tiles: 512 x 256, both accumulators, one load of B.
//     A single tile moves 64 KB of operands per 64-deep k-block into a pair, which at
//     the ~54 bytes a clock that L2 gives an SM takes 596 cycles against its MMAs' 512;
//   * eight epilogue warps that hand the accumulator back as soon as they hold it, and
//     stores through swizzled shared tiles and TMA, which clips ragged edges.
// Tiles run in groups of 16 row tiles, row tiles fastest, so that what the ~74 pairs
// read at one time (about 16 x 5 tiles' operands) stays in L2. Large products run at the
// 1000 W limit, so traffic costs clock. Back to back, groups of 16 against 8, in us at the
// median SM clock: forward of 8192 tokens, d 4096, f 11008: 1621 at 1362 MHz / 1644 at
// 1360; of 4096 tokens 835 at 1357 / 848 at 1392 (4 % fewer clocks); of 8192 tokens,
// d 2048, f 5504: 441 at 1392 / 445 at 1383; backward of 4096 tokens 2327 at 1322 / 2323
// at 1325.
//
// Its grid is persistent: whole tiles in turn, and where the last round would leave
// most pairs idle, that round's tiles are cut along the contraction into equal
// pieces (Sched). A piece writes its FP32 partial to the workspace, and k_ffn_join
// adds a tile's pieces in contraction order and runs the epilogue. (Joining inside
// the kernel, by the piece that arrives last, needs a fence that does not return
// while the SM's TMA loads keep coming: 54.9 us against 49 for 256 tokens, d 4096,
// f 11008.)
//
// k_ffn_skinny (few tokens, kSkinnyTokens): weights are the MMA's M side (128 rows per CTA:
// 64 gate and 64 up rows in the gated forms), tokens its N side (16 ..), so each
// weight is read once and the kernel is a stream over them, bound by HBM. Clusters of
// 1-8 CTAs split the contraction; their FP32 partials are summed over distributed
// shared memory in rank order (no atomics, no workspace).
//
// The kernels of one call follow each other with programmatic dependent launch: the
// next one sets up (and the skinny one requests its first weights, which no kernel
// of the call writes) while the previous one finishes.
//
// Waits are bounded as in mb_gemm.cu: on expiry a CTA raises the device's error word
// (mb_ffn_status), waits (bounded) for its own copies, leaves NaN for the results it
// does not have, frees TMEM and returns. The NaN pass through the call's later kernels
// into its outputs, where the gates of the optimizers find them.
#include <atomic>
#include <mutex>

#include "mb_async.cuh"
#include "mb_common.cuh"
#include "mb_ffn_deal.cuh"
#include "mb_tc.cuh"

namespace mb {

int act_unpack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t d, void* out, int out_dtype,
               int64_t ld, cudaStream_t st);

namespace ffn {

__device__ int32_t g_ffn_err;

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int kFeat = BN / 2;  // features of a gated tile (gate | up halves)
constexpr int kEpiWarps = 8;  // two per TMEM lane quarter, each with half of the tile's columns
constexpr int kPairThreads = 64 + 32 * kEpiWarps;
constexpr int kTileA = BM * BK * 2;         // 16 KiB: this CTA's rows of A
constexpr int kTileB = (BN / 2) * BK * 2;   // 16 KiB: this CTA's half of B
constexpr int kBox = 64 * 64 * 2;           // 8 KiB: one 64 x 64 MN-major box
constexpr int kStoreTile = 32 * 64 * 2;     // 4 KiB: a warp's 32 rows x 64 columns
constexpr int kBarBytes = 512;
constexpr uint32_t kTmemCols = 512;

template <int N> struct Int {
  static constexpr int value = N;
};

// What a product's epilogue does. kPlainF32: FP32 output (dh); kGatedBwd reads a
// 16-bit dh (the caller's), kGatedBwdF32 an FP32 one.
enum Epi { kPlain = 0, kGated = 1, kGatedBwd = 2, kPlainF32 = 3, kGatedBwdF32 = 4 };
constexpr bool is_plain(int epi) { return epi == kPlain || epi == kPlainF32; }
constexpr bool is_bwd(int epi) { return epi == kGatedBwd || epi == kGatedBwdF32; }

// The ring, and shared memory of an epilogue warp: one store tile, or in the
// backward form a 32 x 32 block each of dg, du and h.
constexpr int kOutBlock = 32 * 32 * 2;
constexpr int ring_bytes(int epi) { return (is_bwd(epi) ? 5 : 6) * (kTileA + kTileB); }
constexpr int warp_bytes(int epi) { return is_bwd(epi) ? 3 * kOutBlock : kStoreTile; }
constexpr int pair_smem(int epi) {
  return 1024 + ring_bytes(epi) + kEpiWarps * warp_bytes(epi) + kBarBytes;
}
static_assert(pair_smem(kPlain) <= 232448 && pair_smem(kGatedBwd) <= 232448, "shared memory of one SM");
static_assert(warp_bytes(kGatedBwd) % 512 == 0, "swizzled blocks stay aligned");

constexpr int kMaxMaps = 11;

struct PairMaps {
  CUtensorMap m[kMaxMaps];
};

struct PairArgs : Deal {
  int nmaps;
  int st, stage;  // ring stages and their bytes: A, B and, with pairing 2, the second tile's A
  float* partials;    // workspace of the pieces of cut tiles
  int act;
  int want_h;       // backward: store h
  const void* dh;   // backward input: FP32 (kGatedBwdF32) or 16-bit
  int64_t lddh;
  FaultPlan fault;  // test-only: a tile whose first k-block is withheld, and the launch's wait bound
};

// ------------------------------------------------------------- primitives --

__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// Completes on the barrier at cluster address `bar` (the even CTA's); no multicast.
__device__ __forceinline__ void load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Instruction descriptor (kind::f16): FP32 accumulator, A and B of one 16-bit type
// (bits 7, 10: 1 = BF16), bits 15 / 16 set for an MN-major A / B, N >> 3, M >> 4.
__device__ __forceinline__ uint32_t idesc(bool f16, bool a_mn, bool b_mn, int m, int n) {
  const uint32_t t = f16 ? 0u : 1u;
  return (1u << 4) | (t << 7) | (t << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Shared-memory descriptors of 128-byte-swizzled tiles (layout type 2 at bits
// 61-63, version 1 at bits 46-47), offsets in 16-byte units.
// K-major: rows of 64 elements (128 B), 8-row groups 1024 B apart (SBO); a 16-deep
// slice is 32 B further.
// MN-major: boxes of 64 (MN) x 64 (K), one K index per 128-byte row: 8-K groups
// 1024 B apart (SBO), the next 64 MN elements one box further (LBO); a 16-deep
// slice is 16 rows = 2048 B further.
__device__ __forceinline__ uint64_t desc_at(uint32_t saddr, bool mn) {
  const uint64_t lbo = mn ? (uint64_t)(kBox >> 4) : 1u;
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (lbo << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
constexpr uint32_t desc_slice(bool mn) { return (mn ? 2048u : 32u) >> 4; }

template <bool kMn>
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr, int slice) {
  return desc_at(saddr, kMn) + (uint32_t)slice * desc_slice(kMn);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ------------------------------------------------------------- arithmetic --

// Two FP32 values in a register pair: sm_100 multiplies and adds both at once, which
// halves the epilogues' arithmetic.
struct Two {
  uint64_t v;
};

__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Two two(float x) { return two(x, x); }
__device__ __forceinline__ void split(Two a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// sigma(z) = 1 / (1 + 2^(-z log2 e)); 2^.. of a very negative z is infinite and sigma 0.
__device__ __forceinline__ Two sigmoid(Two z) {
  float x, y;
  split(z * two(-1.4426950408889634f), x, y);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y));
  split(two(x, y) + two(1.0f), x, y);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(y));
  return two(x, y);
}

constexpr float kGeluC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// Past |g| = 64 GELU's sigma(z) is 0 or 1 to the last bit of FP32; stopping there keeps
// g^3 finite, so that z' times a zero is not a NaN.
__device__ __forceinline__ Two gelu_arg(Two g) {
  float x, y;
  split(g, x, y);
  return two(fminf(fmaxf(x, -64.0f), 64.0f), fminf(fmaxf(y, -64.0f), 64.0f));
}

template <int kAct>
__device__ __forceinline__ Two gated(Two g, Two u) {
  Two z = g;
  if constexpr (kAct == MB_ACT_GELU_TANH) {
    const Two c = gelu_arg(g);
    z = c * fma2(c * c, two(kGeluC * kGeluA), two(kGeluC));
  }
  return g * sigmoid(z) * u;
}

// dg, du and h of two elements.
template <int kAct>
__device__ __forceinline__ void gated_bwd(Two g, Two u, Two dh, Two& dg, Two& du, Two& h) {
  Two z = g, zp;
  if constexpr (kAct == MB_ACT_GELU_TANH) {
    const Two c = gelu_arg(g), c2 = c * c;
    z = c * fma2(c2, two(kGeluC * kGeluA), two(kGeluC));
    zp = fma2(c2, two(3.0f * kGeluC * kGeluA), two(kGeluC));
  }
  const Two s = sigmoid(z), a = g * s;
  h = a * u;
  du = dh * a;
  Two slope = fma2(s, two(-1.0f), two(1.0f));  // s + a (1 - s) z'
  if constexpr (kAct == MB_ACT_GELU_TANH) slope = slope * zp;
  dg = dh * u * fma2(a, slope, s);
}

// f(Int<activation>): one copy of a loop for each, with no test inside.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  if (act == MB_ACT_SILU) f(Int<MB_ACT_SILU>{});
  else f(Int<MB_ACT_GELU_TANH>{});
}

template <bool kF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kF16) {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  } else {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
}

template <bool kF16>
__device__ __forceinline__ uint32_t pack2(Two a) {
  float x, y;
  split(a, x, y);
  return pack2<kF16>(x, y);
}

// 16-byte chunk `c` (0..7) of row `r` of a 128-byte-swizzled store tile.
__device__ __forceinline__ uint4* tile_chunk(uint8_t* tile, int r, int c) {
  return reinterpret_cast<uint4*>(tile + r * 128 + ((c ^ (r & 7)) << 4));
}

template <bool kF16>
__device__ __forceinline__ void put_row(uint8_t* tile, int r, int c0, const float* v) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *tile_chunk(tile, r, c0 + c) = make_uint4(pack2<kF16>(v[8 * c], v[8 * c + 1]), pack2<kF16>(v[8 * c + 2], v[8 * c + 3]),
                                              pack2<kF16>(v[8 * c + 4], v[8 * c + 5]), pack2<kF16>(v[8 * c + 6], v[8 * c + 7]));
}

// The same of a 32 x 32 16-bit block (64-byte rows, 64-byte swizzle).
__device__ __forceinline__ uint4* block_chunk(uint8_t* block, int r, int c) {
  return reinterpret_cast<uint4*>(block + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// Four consecutive 16-bit values (8-byte aligned when all four exist).
template <bool kF16>
__device__ __forceinline__ void store_quad(void* p, int64_t e, int n, const float (&v)[4]) {
  uint16_t* o = static_cast<uint16_t*>(p) + e;
  if (n == 4) {
    *reinterpret_cast<uint2*>(o) = make_uint2(pack2<kF16>(v[0], v[1]), pack2<kF16>(v[2], v[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) o[j] = f2h<kF16>(v[j]);
  }
}

// Programmatic dependent launch: let the next kernel of the call set up, and wait
// for everything the previous ones wrote.
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------ pair kernel --

// A warp's partial of a cut tile: its 32 rows x 128 accumulator columns (plain: half
// the tile; gated: 64 features' g, then their u).
constexpr int kWarpCols = BN / 2;
constexpr int kWarpPartial = 32 * kWarpCols;  // floats

// 32 dh values of one row from feature `col` on (zero past the last feature; rows
// are 32-byte aligned in the FP32 form, 16-byte in the caller's 16-bit one).
template <int kEpi, bool kF16>
__device__ __forceinline__ void load_dh(const PairArgs& g, int64_t row, int col, float (&v)[32]) {
  const int M = g.p[0].M, N = g.p[0].N;
  const bool in = row < M;
  if constexpr (kEpi == kGatedBwdF32) {
    const float* p = static_cast<const float*>(g.dh) + row * g.lddh + col;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (in && col + 8 * k < N) {  // the row's pitch covers the whole group of 8
        asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(v[8 * k]), "=f"(v[8 * k + 1]), "=f"(v[8 * k + 2]), "=f"(v[8 * k + 3]), "=f"(v[8 * k + 4]),
                       "=f"(v[8 * k + 5]), "=f"(v[8 * k + 6]), "=f"(v[8 * k + 7])
                     : "l"(p + 8 * k)
                     : "memory");
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * k + e] = 0.0f;
      }
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(g.dh) + row * g.lddh + col;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (in && col + 8 * k + 8 <= N) {
        const uint4 w = *reinterpret_cast<const uint4*>(p + 8 * k);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[8 * k + 2 * e] = h2f<kF16>((uint16_t)(ww[e] & 0xffffu));
          v[8 * k + 2 * e + 1] = h2f<kF16>((uint16_t)(ww[e] >> 16));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * k + e] = in && col + 8 * k + e < N ? h2f<kF16>(p[8 * k + e]) : 0.0f;
      }
    }
  }
}

// A NaN in either 16-bit type and, as a word, in FP32.
constexpr uint32_t kNanWord = 0x7fff7fffu;

// What a warp whose wait expired leaves of a tile: NaN in all outputs that it would have
// written, or in its partial of a cut tile, so that what reads them sees it.
template <int kEpi>
__device__ __noinline__ void store_nan(const PairMaps& maps, const PairArgs& g, int prob, float4* partial, uint8_t* out,
                                       int row0, int col0) {
  const int lane = threadIdx.x & 31;
  const uint4 nan = make_uint4(kNanWord, kNanWord, kNanWord, kNanWord);
  if (partial) {
    for (int i = 0; i < kWarpPartial / 128; ++i) reinterpret_cast<uint4*>(partial)[i * 32] = nan;
    return;
  }
  const Problem& p = g.p[prob];
  if (lane == 0) store_wait_read<0>();
  __syncwarp();
  for (int i = lane; i < warp_bytes(kEpi) / 16; i += 32) reinterpret_cast<uint4*>(out)[i] = nan;
  fence_async();
  __syncwarp();
  if (lane == 0) {
    constexpr int kCols = kEpi == kPlainF32 || is_bwd(kEpi) ? 32 : 64;  // of a store's box
    constexpr int kWide = is_plain(kEpi) ? kWarpCols : kFeat / 2;
    for (int c = 0; c < kWide && col0 + c < p.N; c += kCols) {
      store_2d(&maps.m[p.o], out, col0 + c, row0);
      if constexpr (is_bwd(kEpi)) {
        store_2d(&maps.m[p.o + 1], out, col0 + c, row0);
        if (g.want_h) store_2d(&maps.m[p.o + 2], out, col0 + c, row0);
      }
    }
    store_commit();
  }
}

// kAnyA: A's layout is each problem's; else K-major. kBMn: B stored [K, N].
template <int kEpi, bool kAnyA, bool kBMn, bool kF16>
__global__ void __launch_bounds__(kPairThreads, 1)
    k_ffn_pair(const __grid_constant__ PairMaps maps, const __grid_constant__ PairArgs g) {
  constexpr int kMaxStages = ring_bytes(kEpi) / (kTileA + kTileB);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sOut = ring + ring_bytes(kEpi);
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + kEpiWarps * warp_bytes(kEpi));
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;   // [2]: one arrival per epilogue warp of both CTAs
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int unit = (int)(blockIdx.x >> 1);
  Item item;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2 && lane < g.nmaps) prefetch_map(&maps.m[lane]);
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      pdl_wait();
      // Issuing a stage must stay well under its MMAs' 512 cycles, so everything that an
      // item fixes is out of the loop (two more loads under a run-time condition in it
      // cost the weight gradients 11 %).
      const int st = g.st;
      const uint32_t stage = (uint32_t)g.stage;
      const uint32_t full0 = mapa_u32(smem_u32(full), 0);  // the even CTA's barriers
      const uint32_t ring0 = smem_u32(ring);
      int s = 0, issued = 0;
      uint32_t ph = 0;
      for (Items work(g.sched, unit); !*abort_flag && work.next(g, item);) {
        const Problem& p = g.p[item.prob];
        const int arow = item.bm * 2 * BM + (int)rank * BM;
        // gated tiles: 128 features from gate (even CTA) or up (odd CTA)
        const int brow = is_plain(kEpi) ? item.bn * BN + (int)rank * (BN / 2) : item.bn * kFeat;
        const bool a_mn = kAnyA && p.a_mn;
        const uint32_t bytes = 2 * (item.count * kTileA + kTileB);
        const int seg_kb = p.kb;
        const CUtensorMap* ma = &maps.m[p.a[0]];
        const CUtensorMap* mb_ = &maps.m[p.b[is_plain(kEpi) ? 0 : (int)rank]];
        const CUtensorMap* ma1 = &maps.m[p.a[1]];
        const CUtensorMap* mb1 = &maps.m[p.b[1]];
        const bool withhold = item.tile == g.fault.unit && item.k0 == 0;  // test-only: the MMA warp's wait expires
        int k0 = item.k0 * BK;
        if (is_plain(kEpi) && item.k0 >= seg_kb) {
          ma = ma1;
          mb_ = mb1;
          k0 -= seg_kb * BK;
        }
        auto fill = [&](auto count) {  // one loop each for single and double tiles
          constexpr bool two = decltype(count)::value == 2;
          for (int kb = item.k0; kb < item.k1; ++kb) {
            if (is_plain(kEpi) && kb == seg_kb) {  // the second segment
              ma = ma1;
              mb_ = mb1;
              k0 = 0;
            }
            if (!mbar_wait(&empty[s], ph ^ 1, abort_flag, g.fault.limit_ns)) break;
            if (!withhold || kb > 0) {
              const uint32_t bar = full0 + 8u * (uint32_t)s;
              const uint32_t a = ring0 + (uint32_t)s * stage, b = a + kTileA, a2 = b + kTileB;
              if (leader) mbar_expect_tx(&full[s], bytes);
              if constexpr (kAnyA) {  // 64 x 64 boxes serve both layouts
                load_2d_pair(a, ma, bar, a_mn ? arow : k0, a_mn ? k0 : arow);
                load_2d_pair(a + kBox, ma, bar, a_mn ? arow + 64 : k0, a_mn ? k0 : arow + 64);
                if constexpr (two) {
                  load_2d_pair(a2, ma, bar, a_mn ? arow + 256 : k0, a_mn ? k0 : arow + 256);
                  load_2d_pair(a2 + kBox, ma, bar, a_mn ? arow + 320 : k0, a_mn ? k0 : arow + 320);
                }
              } else {
                load_2d_pair(a, ma, bar, k0, arow);
                if constexpr (two) load_2d_pair(a2, ma, bar, k0, arow + 256);
              }
              if constexpr (kBMn) {
                load_2d_pair(b, mb_, bar, brow, k0);
                load_2d_pair(b + kBox, mb_, bar, brow + 64, k0);
              } else {
                load_2d_pair(b, mb_, bar, k0, brow);
              }
            }
            k0 += BK;
            ++issued;
            if (++s == st) {
              s = 0;
              ph ^= 1;
            }
          }
        };
        if (item.count == 2) fill(Int<2>{});
        else fill(Int<1>{});
      }
      if (*abort_flag && leader) {
        // bounded wait for both CTAs' loads still in flight (they land on the even CTA's barriers)
        const uint64_t t0 = globaltimer();
        for (int k = issued - st > 0 ? issued - st : 0; k < issued; ++k)
          while (!mbar_try_wait(&full[k % st], (k / st) & 1) && globaltimer() - t0 < g.fault.limit_ns) {
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      pdl_wait();  // so that its waits' bounds count from here
      const int st = g.st;
      const uint32_t ring0 = smem_u32(ring), stage16 = (uint32_t)g.stage >> 4;
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (Items work(g.sched, unit); !*abort_flag && work.next(g, item);) {
        const bool a_mn = kAnyA && g.p[item.prob].a_mn;
        const uint32_t id = idesc(kF16, a_mn, kBMn, 2 * BM, BN);
        const uint64_t da0 = desc_at(ring0, a_mn), db0 = desc_at(ring0 + kTileA, kBMn);
        const uint32_t a_slice = desc_slice(a_mn);
        auto slot_free = [&](int i) {
          return mbar_wait_cluster(&acc_empty[i & 1], ((i >> 1) & 1) ^ 1, abort_flag, g.fault.limit_ns);
        };
        auto stage_here = [&] { return mbar_wait(&full[s], ph, abort_flag, g.fault.limit_ns); };
        // stage s into accumulator slot i: tile m's A against B
        auto multiply = [&](int stage, int m, int i, bool first) {
          const uint32_t off = (uint32_t)stage * stage16;
          const uint64_t da = da0 + off + (m == 0 ? 0 : (kTileA + kTileB) >> 4), db = db0 + off;
          const uint32_t acc = tmem + (uint32_t)((i & 1) * BN);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma_pair(acc, da + (uint32_t)k * a_slice, db + (uint32_t)k * desc_slice(kBMn), id,
                      first && k == 0 ? 0u : 1u);
        };
        auto advance = [&] {
          if (++s == st) {
            s = 0;
            ph ^= 1;
          }
        };
        const int n = item.k1 - item.k0;
        if (!slot_free(it)) break;
        tc_fence_after();
        bool good = true;
        if (item.count == 1) {
          for (int kb = 0; kb < n; ++kb) {
            if (!(good = stage_here())) break;
            tc_fence_after();
            multiply(s, 0, it, kb == 0);
            umma_commit_both(&empty[s]);
            advance();
          }
          // an aborted tile is not handed over: the odd CTA cannot see this CTA's abort flag
          if (good) umma_commit_both(&acc_full[it & 1]);
        } else {
          // two tiles on the same B, stage by stage
          for (int kb = 0; kb < n; ++kb) {
            if (!(good = stage_here())) break;
            tc_fence_after();
            multiply(s, 0, it, kb == 0);
            if (kb + 1 == n) umma_commit_both(&acc_full[it & 1]);
            if (kb == 0) {  // the first tile starts while the epilogue still drains the second accumulator
              if (!(good = slot_free(it + 1))) break;
              tc_fence_after();
            }
            multiply(s, 1, it + 1, kb == 0);
            umma_commit_both(&empty[s]);
            advance();
          }
          if (good) umma_commit_both(&acc_full[(it + 1) & 1]);
        }
        if (!good) break;
        it += item.count;
      }
      if (*abort_flag) {
        umma_commit_pair(drain);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(drain, 0) && globaltimer() - t0 < g.fault.limit_ns) {
        }
      }
    }
  } else {
    const int q = warp & 3;              // TMEM lane quarter this warp may read
    const int half = (warp - 2) >> 2;    // its half of the tile's columns (gated: features)
    const int w16 = (int)rank * kEpiWarps + half * 4 + q;
    uint8_t* out = sOut + (warp - 2) * warp_bytes(kEpi);
    int it = 0, ok = 1;
    pdl_wait();
    // a cut tile's partial of this warp: float4 j of lane l at j * 32 + l
    auto my_partial = [&](const Item& it) {
      return reinterpret_cast<float4*>(g.partials) +
             ((int64_t)(it.tile * g.sched.ways + it.piece) * 2 * kEpiWarps + w16) * (kWarpPartial / 4) + lane;
    };
    Items work(g.sched, unit);
    int m = 0;
    item.count = 0;
    while (true) {
      if (m == item.count) {  // the next item's first tile, or this item's second
        if (!work.next(g, item)) break;
        m = 0;
      }
      const int a = it & 1;
      const uint32_t use = it >> 1;
      ++it;
      const Problem& p = g.p[item.prob];
      const int row0 = (item.bm + m) * 2 * BM + (int)rank * BM + q * 32;
      ++m;
      const int col0 = is_plain(kEpi) ? item.bn * BN + half * kWarpCols : item.bn * kFeat + half * (kFeat / 2);
      const bool in = row0 < p.M && col0 < p.N;  // some of this warp's outputs exist
      float dh[32];
      if constexpr (is_bwd(kEpi)) {
        if (in) load_dh<kEpi, kF16>(g, row0 + lane, col0, dh);  // arrives while the MMAs run
      }
      if (ok && lane == 0) ok = mbar_wait(&acc_full[a], use & 1, abort_flag, g.fault.limit_ns) && !*abort_flag;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) {  // this tile and the unit's others will not come: NaN stands for them
        if (in) store_nan<kEpi>(maps, g, item.prob, item.piece >= 0 ? my_partial(item) : nullptr, out, row0, col0);
        continue;
      }
      tc_fence_after();
      // this warp's accumulator columns: plain 0..127 from here; gated g at 0..63, u at kFeat..
      const uint32_t acc = tmem + (uint32_t)(a * BN) + ((uint32_t)(q * 32) << 16) +
                           (uint32_t)(half * (is_plain(kEpi) ? kWarpCols : kFeat / 2));
      // 32 accumulator columns: block b (0..3) of this warp's 128
      auto fetch = [&](int b, float* v) {
        uint32_t r[32];
        tmem_ld32(acc + (uint32_t)(is_plain(kEpi) ? 32 * b : 32 * (b & 1) + kFeat * (b >> 1)), r);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
      };
      // hand the accumulator back: every lane's loads of it are complete
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[a]), 0));
      };
      if (!in) {
        release();
      } else if (item.piece >= 0) {
        float4* mine = my_partial(item);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float v[32];
          fetch(b, v);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mine[(b * 8 + k) * 32] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        }
        release();
      } else {
        if constexpr (kEpi == kPlainF32) {
          float v[128];
#pragma unroll
          for (int b = 0; b < 4; ++b) fetch(b, v + 32 * b);
          release();
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if (col0 + 32 * b >= p.N) break;  // warp-uniform
            if (lane == 0) store_wait_read<0>();  // the store before has read this tile
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float* x = v + 32 * b + 4 * k;
              *tile_chunk(out, lane, k) =
                  make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
            }
            fence_async();
            __syncwarp();
            if (lane == 0) {
              store_2d(&maps.m[p.o], out, col0 + 32 * b, row0);
              store_commit();
            }
          }
        } else if constexpr (kEpi == kPlain) {
          uint32_t w[4][16];  // the warp's 128 columns, rounded
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            float v[32];
            fetch(b, v);
#pragma unroll
            for (int k = 0; k < 16; ++k) w[b][k] = pack2<kF16>(v[2 * k], v[2 * k + 1]);
          }
          release();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (col0 + 64 * h >= p.N) break;  // warp-uniform
            if (lane == 0) store_wait_read<0>();  // the store before has read this tile
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint32_t* x = w[2 * h + c / 4] + 4 * (c % 4);
              *tile_chunk(out, lane, c) = make_uint4(x[0], x[1], x[2], x[3]);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) {
              store_2d(&maps.m[p.o], out, col0 + 64 * h, row0);
              store_commit();
            }
          }
        } else if constexpr (kEpi == kGated) {
          if (lane == 0) store_wait_read<0>();  // the tile before has been read out
          __syncwarp();
#pragma unroll 1
          for (int b = 0; b < 2; ++b) {
            float v[64];
            fetch(b, v);
            fetch(b + 2, v + 32);
            if (b == 1) release();
            with_act(g.act, [&](auto act) {
#pragma unroll
              for (int j = 0; j < 32; j += 2)
                split(gated<decltype(act)::value>(two(v[j], v[j + 1]), two(v[32 + j], v[33 + j])), v[j], v[j + 1]);
            });
            put_row<kF16>(out, lane, 4 * b, v);
          }
          fence_async();
          __syncwarp();
          if (lane == 0) {
            store_2d(&maps.m[p.o], out, col0, row0);
            store_commit();
          }
        } else {
          uint8_t* tdg = out;
          uint8_t* tdu = tdg + kOutBlock;
          uint8_t* th = tdu + kOutBlock;
#pragma unroll 1
          for (int b = 0; b < 2; ++b) {
            const bool last = b == 1 || col0 + 32 >= p.N;  // warp-uniform
            float v[64];
            fetch(b, v);
            fetch(b + 2, v + 32);
            if (last) release();
            if (lane == 0) store_wait_read<0>();  // the block before has been read out
            __syncwarp();
            with_act(g.act, [&](auto act) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {  // 8 features each
                uint32_t og[4], ou[4], oh[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int j = k * 8 + i * 2;
                  Two dg, du, h;
                  gated_bwd<decltype(act)::value>(two(v[j], v[j + 1]), two(v[32 + j], v[33 + j]), two(dh[j], dh[j + 1]),
                                                  dg, du, h);
                  og[i] = pack2<kF16>(dg);
                  ou[i] = pack2<kF16>(du);
                  oh[i] = pack2<kF16>(h);
                }
                *block_chunk(tdg, lane, k) = make_uint4(og[0], og[1], og[2], og[3]);
                *block_chunk(tdu, lane, k) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
                *block_chunk(th, lane, k) = make_uint4(oh[0], oh[1], oh[2], oh[3]);
              }
            });
            if (!last) load_dh<kEpi, kF16>(g, row0 + lane, col0 + 32, dh);
            fence_async();
            __syncwarp();
            if (lane == 0) {
              const int col = col0 + 32 * b;
              store_2d(&maps.m[p.o], tdg, col, row0);
              store_2d(&maps.m[p.o + 1], tdu, col, row0);
              if (g.want_h) store_2d(&maps.m[p.o + 2], th, col, row0);
              store_commit();
            }
            if (last) break;
          }
        }
      }
    }
    if (lane == 0) store_wait_read<0>();  // the stores have read their tiles; the kernel's end completes them
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync();  // after every bounded wait of both CTAs
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_ffn_err, 1);
}

// Completes the cut tiles of a pair launch: adds each one's pieces in contraction
// order and runs the product's epilogue. A warp takes 16 rows x 16 columns (features), a
// lane a row's 8: it reads 256 contiguous bytes of a piece at a time, all of a thread's
// loads in flight at once, and writes whole sectors. A CTA's warps take different rows
// of the tile, so that those past the last token are spread evenly.
// Gated, d 4096, f 11008: 256 tokens 58.0 -> 53.7 us against 32 rows x 16 columns a warp
// with one piece's loads in flight at a time; f 4736: 28.8 -> 27.
struct JoinArgs {
  PairArgs g;
  void* o[kMaxProblems];  // of each problem; of the backward form: dg, du, h
  int64_t ldo[kMaxProblems];
};

// What an SM has left beside a pair kernel's CTA (registers, 1.5 KB of shared memory) takes
// one CTA of this many threads, which is there when the pair kernel ends: 0.5 us less
// than CTAs of 128.
constexpr int join_threads(int epi) { return epi == kGated ? 384 : is_bwd(epi) ? 192 : 256; }
constexpr int kJoinCols = 8;

// kJoinCols 16-bit values from element e on, the first n of them (rows are 16-byte
// aligned and kJoinCols divides e's column).
template <bool kF16>
__device__ __forceinline__ void store_cols(void* p, int64_t e, int n, const float (&v)[kJoinCols]) {
  uint16_t* o = static_cast<uint16_t*>(p) + e;
  if (n == kJoinCols) {
#pragma unroll
    for (int h = 0; h < kJoinCols / 8; ++h)
      reinterpret_cast<uint4*>(o)[h] =
          make_uint4(pack2<kF16>(v[8 * h], v[8 * h + 1]), pack2<kF16>(v[8 * h + 2], v[8 * h + 3]),
                     pack2<kF16>(v[8 * h + 4], v[8 * h + 5]), pack2<kF16>(v[8 * h + 6], v[8 * h + 7]));
  } else {
#pragma unroll
    for (int j = 0; j < kJoinCols; ++j)
      if (j < n) o[j] = f2h<kF16>(v[j]);
  }
}

// volatile, so that a thread's loads are all issued before it adds
__device__ __forceinline__ float4 ld_partial(const float4* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

template <int kEpi, bool kF16>
__global__ void __launch_bounds__(join_threads(kEpi)) k_ffn_join(const __grid_constant__ JoinArgs j) {
  pdl_trigger();
  const PairArgs& g = j.g;
  constexpr int kGroups = (is_plain(kEpi) ? kWarpCols : kFeat / 2) / kJoinCols;  // of a piece's warp
  constexpr int kParts = is_plain(kEpi) ? 1 : 2;                                 // value, or g and u
  const int item = (int)(blockIdx.x * (join_threads(kEpi) / 32) + (threadIdx.x >> 5));
  const int w16 = item % (2 * kEpiWarps), g0 = item / (2 * kEpiWarps) % kGroups;
  const int lane = (g0 & 1) * 16 + (threadIdx.x & 15);  // of the pieces' warp: its row
  const int group = (g0 & ~1) + ((threadIdx.x >> 4) & 1);
  Item it;
  it.tile = item / kGroups / (2 * kEpiWarps);
  it.count = 1;
  if (it.tile >= g.sched.long_tiles || !place_tile(g, it)) return;
  const Problem& p0 = g.p[it.prob];
  const int out = is_plain(kEpi) ? it.prob : 0;
  const int half = (w16 & (kEpiWarps - 1)) >> 2;
  const int64_t row = (int64_t)it.bm * 2 * BM + w16 / kEpiWarps * BM + (w16 & 3) * 32 + lane;
  const int col =
      (is_plain(kEpi) ? it.bn * BN + half * kWarpCols : it.bn * kFeat + half * (kFeat / 2)) + kJoinCols * group;
  if (row >= p0.M || col >= p0.N) return;
  const int n = p0.N - col < kJoinCols ? p0.N - col : kJoinCols;
  pdl_wait();
  const float4* src = reinterpret_cast<const float4*>(g.partials) +
                      ((int64_t)it.tile * g.sched.ways * 2 * kEpiWarps + w16) * (kWarpPartial / 4) +
                      group * (kJoinCols / 4) * 32 + lane;
  constexpr int64_t kPiece = (int64_t)2 * kEpiWarps * kWarpPartial / 4;
  float v[kParts][kJoinCols];
  auto add = [&](auto ways) {
    float4 x[decltype(ways)::value][kParts][kJoinCols / 4];
#pragma unroll
    for (int i = 0; i < decltype(ways)::value; ++i)
#pragma unroll
      for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int c = 0; c < kJoinCols / 4; ++c)
          x[i][p][c] = ld_partial(src + i * kPiece + (p * (kFeat / 2) / 4 + c) * 32);
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
      for (int c = 0; c < kJoinCols / 4; ++c) {
        float4 t = x[0][p][c];
#pragma unroll
        for (int i = 1; i < decltype(ways)::value; ++i) {
          t.x += x[i][p][c].x; t.y += x[i][p][c].y; t.z += x[i][p][c].z; t.w += x[i][p][c].w;
        }
        v[p][4 * c] = t.x; v[p][4 * c + 1] = t.y; v[p][4 * c + 2] = t.z; v[p][4 * c + 3] = t.w;
      }
  };
  static_assert(kMaxWays == 4);
  if (g.sched.ways == 2) add(std::integral_constant<int, 2>{});
  else if (g.sched.ways == 3) add(std::integral_constant<int, 3>{});
  else add(std::integral_constant<int, 4>{});
  if constexpr (kEpi == kPlain) {
    store_cols<kF16>(j.o[out], row * j.ldo[out] + col, n, v[0]);
  } else if constexpr (kEpi == kPlainF32) {
    float* o = static_cast<float*>(j.o[out]) + row * j.ldo[out] + col;
#pragma unroll
    for (int c = 0; c < kJoinCols; c += 4) {
      if (c + 4 <= n) {
        *reinterpret_cast<float4*>(o + c) = make_float4(v[0][c], v[0][c + 1], v[0][c + 2], v[0][c + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < n) o[c + e] = v[0][c + e];
      }
    }
  } else if constexpr (kEpi == kGated) {
    with_act(g.act, [&](auto act) {
#pragma unroll
      for (int c = 0; c < kJoinCols; c += 2)
        split(gated<decltype(act)::value>(two(v[0][c], v[0][c + 1]), two(v[1][c], v[1][c + 1])), v[0][c], v[0][c + 1]);
    });
    store_cols<kF16>(j.o[0], row * j.ldo[0] + col, n, v[0]);
  } else {
    float dg[kJoinCols], du[kJoinCols], h[kJoinCols], dh[kJoinCols];
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c) {
      dh[c] = 0.0f;
      if (c < n) {
        if constexpr (kEpi == kGatedBwdF32) dh[c] = static_cast<const float*>(g.dh)[row * g.lddh + col + c];
        else dh[c] = h2f<kF16>(static_cast<const uint16_t*>(g.dh)[row * g.lddh + col + c]);
      }
    }
    with_act(g.act, [&](auto act) {
#pragma unroll
      for (int c = 0; c < kJoinCols; c += 2) {
        Two a, b, e;
        gated_bwd<decltype(act)::value>(two(v[0][c], v[0][c + 1]), two(v[1][c], v[1][c + 1]), two(dh[c], dh[c + 1]), a,
                                        b, e);
        split(a, dg[c], dg[c + 1]);
        split(b, du[c], du[c + 1]);
        split(e, h[c], h[c + 1]);
      }
    });
    store_cols<kF16>(j.o[0], row * j.ldo[0] + col, n, dg);
    store_cols<kF16>(j.o[1], row * j.ldo[1] + col, n, du);
    if (g.want_h) store_cols<kF16>(j.o[2], row * j.ldo[2] + col, n, h);
  }
}

// ---------------------------------------------------------- skinny kernel --

struct Maps {
  CUtensorMap a[2], b[2];  // weights (K segments, or gate and up), tokens
};

constexpr int kSkinnyThreads = 128;
constexpr int kSkinnyPitch = 132;  // floats between tokens' 128 partials in shared memory

struct SkinnyArgs {
  int tokens;     // M of the product
  int n;          // tokens padded to a multiple of 16 (MMA N)
  int rows;       // output features
  int kb, nseg;   // 64-deep blocks of one K segment; segments
  int split;      // cluster CTAs sharing one tile's contraction
  int st;         // ring stages
  int act;
  uint32_t tmem_cols;
  void* o0;       // plain / gated output, or dg
  void* o1;       // du
  void* o2;       // h (or null)
  const void* dh;  // FP32 (kGatedBwdF32) or 16-bit
  int64_t ldo, ldu, ldh, lddh;
  FaultPlan fault;  // test-only: a CTA whose first k-block is withheld, and the launch's wait bound
};

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <int kEpi, bool kAMn, bool kF16>
__global__ void __launch_bounds__(kSkinnyThreads) k_ffn_skinny(const __grid_constant__ Maps maps, const SkinnyArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tile_b = g.n * BK * 2;  // a multiple of 2048: every tile stays 1024-byte aligned
  uint8_t* sA = smem;
  uint8_t* sB = sA + g.st * kTileA;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + g.st * tile_b);
  uint64_t* empty = full + g.st;
  uint64_t* acc_full = empty + g.st;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = g.split > 1 ? (int)cluster_rank() : 0;
  const int tile = (int)blockIdx.x / g.split;
  const int KB = g.kb * g.nseg;
  const int k_lo = (int)((int64_t)KB * rank / g.split), k_hi = (int)((int64_t)KB * (rank + 1) / g.split);
  const int feat0 = tile * (is_plain(kEpi) ? 128 : 64);

  const bool withhold = (int)blockIdx.x == g.fault.unit;  // test-only; the MMA thread's wait expires
  auto load_weights = [&](int s, int k) {
    const int seg = k >= g.kb ? 1 : 0, k0 = (k - seg * g.kb) * BK;
    mbar_expect_tx(&full[s], kTileA + tile_b);
    uint8_t* a = sA + s * kTileA;
    if constexpr (kAMn) {
      load_2d(a, &maps.a[seg], &full[s], feat0, k0);
      load_2d(a + kBox, &maps.a[seg], &full[s], feat0 + 64, k0);
    } else if constexpr (is_plain(kEpi)) {
      load_2d(a, &maps.a[seg], &full[s], k0, feat0);
    } else {  // 64 gate rows, then the same 64 up rows
      load_2d(a, &maps.a[0], &full[s], k0, feat0);
      load_2d(a + kBox, &maps.a[1], &full[s], k0, feat0);
    }
  };
  auto load_tokens = [&](int s, int k) {
    const int seg = k >= g.kb ? 1 : 0;
    load_2d(sB + s * tile_b, &maps.b[seg], &full[s], (k - seg * g.kb) * BK, 0);
  };
  const int head = k_hi - k_lo < g.st ? k_hi - k_lo : g.st;

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.st; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
    // the ring's first round: weights before anything else is set up, tokens when the
    // kernels before have written them
    for (int i = withhold ? 1 : 0; i < head; ++i) load_weights(i, k_lo + i);
  }
  if (warp == 2 && lane < 4) prefetch_map(lane < 2 ? &maps.a[lane] : &maps.b[lane - 2]);
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(g.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();

  if (warp == 0 && lane == 0) {
    pdl_wait();
    int kit = 0;
    for (int k = k_lo; k < k_hi; ++k, ++kit) {
      const int s = kit % g.st;
      if (kit >= head) {
        if (!mbar_wait(&empty[s], ((kit / g.st) & 1) ^ 1, abort_flag, g.fault.limit_ns)) break;
        load_weights(s, k);
      } else if (withhold && kit == 0) {
        continue;
      }
      load_tokens(s, k);
    }
    if (*abort_flag) {  // bounded wait for this CTA's loads in flight
      const uint64_t t0 = globaltimer();
      for (int k = kit - g.st > 0 ? kit - g.st : 0; k < kit; ++k)
        while (!mbar_try_wait(&full[k % g.st], (k / g.st) & 1) && globaltimer() - t0 < g.fault.limit_ns) {
        }
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t id = idesc(kF16, kAMn, false, 128, g.n);
    pdl_wait();  // so that its waits' bounds count from here
    int kit = 0;
    for (int k = k_lo; k < k_hi; ++k, ++kit) {
      const int s = kit % g.st;
      if (!mbar_wait(&full[s], (kit / g.st) & 1, abort_flag, g.fault.limit_ns)) break;
      tc_fence_after();
      const uint32_t a0 = smem_u32(sA + s * kTileA), b0 = smem_u32(sB + s * tile_b);
#pragma unroll
      for (int i = 0; i < BK / 16; ++i)
        umma_16(tmem, tile_desc<kAMn>(a0, i), tile_desc<false>(b0, i), id, (kit | i) != 0 ? 1u : 0u);
      umma_commit(&empty[s]);
    }
    umma_commit(acc_full);  // also on abort: completion of every MMA issued
  }
  __syncwarp();
  pdl_wait();  // before the first access to what the kernels before may write or read
  // Every thread waits for the last MMA: then the ring is idle and its memory holds
  // the partials. An aborting CTA's are NaN, and so is what the cluster makes of them.
  mbar_wait(acc_full, 0, abort_flag, g.fault.limit_ns);
  if (*abort_flag) {
    const uint64_t t0 = globaltimer();
    while (!mbar_try_wait(acc_full, 0) && globaltimer() - t0 < g.fault.limit_ns) {
    }
  }
  __syncthreads();  // the producer's and the MMA thread's waits have ended too
  tc_fence_after();
  float* part = reinterpret_cast<float*>(smem);
  for (int c = 0; c < g.tokens; c += 16) {
    uint32_t r[16];
    tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)c, r);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c + j < g.tokens) part[(c + j) * kSkinnyPitch + warp * 32 + lane] = __uint_as_float(r[j]);
  }
  if (*abort_flag)  // outside the loop: chosen inside it, 100 tokens, d 1024, f 2816 take 20.4 us for 18.7
    for (int c = 0; c < g.tokens; ++c) part[c * kSkinnyPitch + warp * 32 + lane] = __uint_as_float(kNanWord);
  // The columns go back before the wait for the cluster: a CTA that held them there while
  // its peer waits for columns of another stream's kernel, whose own pair waits for these,
  // would wait for good.
  tc_fence_before();
  if (g.split > 1) cluster_arrive();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols) : "memory");
  }
  if (g.split > 1) cluster_wait();
  // the tile's (token, 4 features) groups, dealt to the cluster's threads; a group's
  // partials are added in rank order
  constexpr int kPer = is_plain(kEpi) ? 32 : 16;
  const int items = g.tokens * kPer;
  const uint32_t base = smem_u32(part);
  for (int i = rank * kSkinnyThreads + (int)threadIdx.x; i < items; i += g.split * kSkinnyThreads) {
    const int j = i / kPer, f4 = (i % kPer) * 4;
    const int64_t tok = j, col = feat0 + f4;
    const int n = g.rows - (feat0 + f4) < 4 ? g.rows - (feat0 + f4) : 4;
    if (n <= 0) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, w[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t at = base + (uint32_t)(j * kSkinnyPitch + f4) * 4u;
#pragma unroll 4
    for (int r = 0; r < g.split; ++r) {
      const uint32_t p = g.split > 1 ? mapa_u32(at, (uint32_t)r) : at;
      const float4 x = ld_cluster_f32x4(p);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      if constexpr (!is_plain(kEpi)) {
        const float4 y = ld_cluster_f32x4(p + 64 * 4);
        w[0] += y.x; w[1] += y.y; w[2] += y.z; w[3] += y.w;
      }
    }
    if constexpr (kEpi == kPlain) {
      store_quad<kF16>(g.o0, tok * g.ldo + col, n, v);
    } else if constexpr (kEpi == kPlainF32) {
      float* o = static_cast<float*>(g.o0) + tok * g.ldo + col;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) o[e] = v[e];
    } else if constexpr (kEpi == kGated) {
      with_act(g.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 4; e += 2)
          split(gated<decltype(act)::value>(two(v[e], v[e + 1]), two(w[e], w[e + 1])), v[e], v[e + 1]);
      });
      store_quad<kF16>(g.o0, tok * g.ldo + col, n, v);
    } else {
      float dg[4], du[4], h[4], dh[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dh[e] = 0.0f;
        if (e < n) {
          if constexpr (kEpi == kGatedBwdF32) dh[e] = static_cast<const float*>(g.dh)[tok * g.lddh + col + e];
          else dh[e] = h2f<kF16>(static_cast<const uint16_t*>(g.dh)[tok * g.lddh + col + e]);
        }
      }
      with_act(g.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          Two a, b, c;
          gated_bwd<decltype(act)::value>(two(v[e], v[e + 1]), two(w[e], w[e + 1]), two(dh[e], dh[e + 1]), a, b, c);
          split(a, dg[e], dg[e + 1]);
          split(b, du[e], du[e + 1]);
          split(c, h[e], h[e + 1]);
        }
      });
      store_quad<kF16>(g.o0, tok * g.ldo + col, n, dg);
      store_quad<kF16>(g.o1, tok * g.ldu + col, n, du);
      if (g.o2 != nullptr) store_quad<kF16>(g.o2, tok * g.ldh + col, n, h);
    }
  }
  if (g.split > 1) cluster_sync();  // no CTA leaves while a peer reads its partials
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_ffn_err, 1);
}

// -------------------------------------------------------------- alignment --

// TMA takes rows that start on 16 bytes. A call's matrices whose rows do not are
// copied to (outputs: from) padded rows of the workspace, all in one launch: a warp a
// row, consecutive lanes consecutive elements.
struct CopyJob {
  const uint16_t* src;
  uint16_t* dst;
  int64_t src_ld, dst_ld, rows, cols;
};

constexpr int kMaxCopies = 5;  // x, gate, up, down, dy; or the four gradients

struct CopyJobs {
  CopyJob j[kMaxCopies];
};

constexpr int kCopyThreads = 256;

__global__ void __launch_bounds__(kCopyThreads) k_ffn_copy(const __grid_constant__ CopyJobs jobs) {
  const CopyJob& j = jobs.j[blockIdx.y];
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kCopyThreads / 32);
  for (int64_t row = (int64_t)blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); row < j.rows; row += warps) {
    const uint16_t* src = j.src + row * j.src_ld;
    uint16_t* dst = j.dst + row * j.dst_ld;
    for (int64_t c = lane; c < j.cols; c += 32 * 8) {
      uint16_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + 32 * i < j.cols) v[i] = src[c + 32 * i];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + 32 * i < j.cols) dst[c + 32 * i] = v[i];
    }
  }
}

// ------------------------------------------------------------------ host --

// 2-D tensor [rows][cols] of `type`, row pitch ld (elements); boxes of 64 or 128
// bytes a row, swizzled over that span.
bool map_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t rows, int64_t cols, int64_t ld,
            int box_cols, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const int elem = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * elem)};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            box_cols * elem == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A matrix in memory (16-bit; dh inside the backward pass: FP32).
struct Mat {
  const void* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
};

// One contraction: out = sum over segments of A B^T, or the gated forms of it.
struct Product {
  int epi = kPlain;
  bool a_mn = false, b_mn = false;  // operand stored [K, M] / [K, N]
  int nseg = 1;
  Mat a[2], b[2];    // gated: a[0] = x, b = gate, up
  Mat o[3];          // outputs (backward: dg, du, h or null)
  Mat dh;
  int64_t M = 0, N = 0, K = 0;  // N: features of a gated form
  int act = 0;

  int64_t kblocks() const { return (K + BK - 1) / BK * nseg; }
};

constexpr int kMaxDevices = 64;
// Longest contraction, in k-blocks (1.3e8 elements): a tile's MMAs then end well inside
// the 2 s that its epilogue waits for them.
constexpr int64_t kMaxKb = (int64_t)1 << 21;

struct KernelEntry {
  std::once_flag once[kMaxDevices];
  int rc[kMaxDevices];
  int pairs[kMaxDevices];
};

int current_device(int* sms) {
  static std::atomic<int> count[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -1;
  // a thread that has made no call of the runtime yet (autograd's, say) has no context,
  // and the tensor-map encoder is a driver call
  static thread_local int bound = -1;
  if (bound != dev) {
    if (cudaSetDevice(dev) != cudaSuccess) return -1;
    bound = dev;
  }
  int n = count[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return -1;
    count[dev].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return dev;
}

// What the products of one call share.
struct Ctx {
  cudaStream_t stream;
  float* partials;  // pair products: the pieces of cut tiles
  bool chained;     // the kernel before on the stream belongs to this call
};

cudaLaunchConfig_t launch_config(cudaLaunchAttribute (&at)[2], int grid, int threads, int smem, int cluster,
                                 const Ctx* ctx) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = ctx ? ctx->stream : nullptr;
  cfg.attrs = at;
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    at[cfg.numAttrs].val.clusterDim.y = 1;
    at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (ctx && ctx->chained) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cfg;
}

// Tokens up to which the weight-streaming kernel runs. Past it the pair kernel's one row
// tile holds all tokens and moves each weight as often, with more tokens to a load. The
// gated forms, against the pair kernel, in us (up to 64 tokens three of its CTAs share an
// SM, from 65 on two):
//   tokens              65            100            128            144
//   d 4096, f 11008     38.6 / 45.1   42.0 / 49.0    45.2 / 49.3    46.3 / 49.2
//   d 2048, f 5504      14.7 / 16.7   16.1 / 16.2    16.8 / 16.3    17.4 / 16.2
//   d 1024, f 2816       9.1 / 11.0   10.6 / 11.3    11.8 / 11.3    12.4 / 11.3
//   d 1200, f 8000      11.8 / 12.4   13.7 / 12.5    14.9 / 12.7    15.8 / 12.6
// so 128 is between the wide blocks' limit and the narrow ones', which is about 100. The
// plain forms: 160 tokens, d 4096, f 11008: 25.5 / 30.0, d 1024, f 2816: 11.1 / 11.4; 192
// tokens, d 2048, f 5504: 27.7 / 15.6.
constexpr int64_t kSkinnyTokens = 128, kSkinnyTokensPlain = 160;
constexpr size_t kJoinBytes = (size_t)kMaxPairs * 2 * kEpiWarps * kWarpPartial * 4;  // one piece a pair

// The workspace's joining part; a forward call whose products are all skinny has none.
size_t join_bytes(int64_t tokens) { return tokens <= kSkinnyTokens ? 0 : kJoinBytes; }

// The launch's maps: one for every matrix and box.
struct MapSet {
  struct Key {
    Mat x;
    int box_cols, box_rows;
  };
  PairMaps maps;
  Key keys[kMaxMaps];
  int n = 0;
  bool ok = true;

  int add(CUtensorMapDataType type, const Mat& x, int box_cols, int box_rows) {
    for (int i = 0; i < n; ++i) {
      const Key& k = keys[i];
      if (k.x.p == x.p && k.x.rows == x.rows && k.x.cols == x.cols && k.x.ld == x.ld && k.box_cols == box_cols &&
          k.box_rows == box_rows)
        return i;
    }
    if (n == kMaxMaps) {
      ok = false;
      return 0;
    }
    keys[n] = {x, box_cols, box_rows};
    ok = ok && map_2d(&maps.m[n], type, x.p, x.rows, x.cols, x.ld, box_cols, box_rows);
    return n++;
  }
};

// `n` products of one kind in one launch; more than one only in the kAnyA form, by
// falling contraction.
template <int kEpi, bool kAnyA, bool kBMn, bool kF16>
int launch_pair(const Product* qs, int n, Ctx& ctx) {
  auto kernel = &k_ffn_pair<kEpi, kAnyA, kBMn, kF16>;
  constexpr int smem = pair_smem(kEpi);
  constexpr CUtensorMapDataType t16 = kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  constexpr CUtensorMapDataType t32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  static KernelEntry entry;  // of this instantiation
  int sms = 0;
  const int dev = current_device(&sms);
  if (dev < 0) return MB_ERR_CUDA;
  std::call_once(entry.once[dev], [&] {
    entry.rc[dev] = MB_ERR_CUDA;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return;
    cudaLaunchAttribute at[2];
    cudaLaunchConfig_t occ = launch_config(at, 2 * (sms / 2), kPairThreads, smem, 2, nullptr);
    int c = 0;
    if (cudaOccupancyMaxActiveClusters(&c, kernel, &occ) != cudaSuccess || c <= 0) return;
    entry.pairs[dev] = c < kMaxPairs ? c : kMaxPairs;
    entry.rc[dev] = MB_OK;
  });
  if (entry.rc[dev] != MB_OK) return entry.rc[dev];
  MapSet maps;
  PairArgs g{};
  int64_t tiles = 0;
  for (int i = 0; i < n; ++i) {
    const Product& q = qs[i];
    Problem& p = g.p[i];
    p.M = (int)q.M; p.N = (int)q.N;
    p.nseg = q.nseg;
    p.a_mn = q.a_mn ? 1 : 0;
    const int64_t cols = is_plain(kEpi) ? BN : kFeat;
    const int64_t mt = (q.M + 2 * BM - 1) / (2 * BM), nt = (q.N + cols - 1) / cols;
    tiles += mt * nt;
    if (tiles > ((int64_t)1 << 29)) return MB_ERR_TOO_LARGE;
    if (q.kblocks() > kMaxKb) return MB_ERR_TOO_LARGE;
    p.kb = (int)((q.K + BK - 1) / BK);
    p.mt = (int)mt; p.nt = (int)nt;
    const int nb = is_plain(kEpi) ? q.nseg : 2;
    for (int k = 0; k < q.nseg; ++k) p.a[k] = maps.add(t16, q.a[k], 64, kAnyA ? 64 : BM);
    for (int k = 0; k < nb; ++k) p.b[k] = maps.add(t16, q.b[k], 64, kBMn ? 64 : BN / 2);
  }
  constexpr bool f32_out = kEpi == kPlainF32;
  for (int i = 0; i < n; ++i)
    for (int k = 0; k < 3; ++k) {
      if (!qs[i].o[k].p) continue;
      const int m = maps.add(f32_out ? t32 : t16, qs[i].o[k], f32_out || is_bwd(kEpi) ? 32 : 64, 32);
      if (k == 0) g.p[i].o = m;
    }
  if (!maps.ok) return MB_ERR_CUDA;
  const Product& q = qs[0];
  const int most = entry.pairs[dev];
  g.nprob = n;
  deal_tiles(g, !is_bwd(kEpi), most);
  const int pairing = g.sched.pairing;
  g.stage = pairing * kTileA + kTileB;
  g.st = ring_bytes(kEpi) / g.stage;
  g.nmaps = maps.n;
  g.act = q.act; g.want_h = q.o[2].p != nullptr;
  g.dh = q.dh.p; g.lddh = q.dh.ld;
  take_fault(kFaultFfn, &g.fault.unit, &g.fault.limit_ns);
  g.partials = ctx.partials;
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t cfg = launch_config(at, 2 * g.sched.units, kPairThreads, smem, 2, &ctx);
  if (cudaLaunchKernelEx(&cfg, kernel, maps.maps, g) != cudaSuccess) return MB_ERR_CUDA;
  ctx.chained = true;
  if (g.sched.ways == 1) return MB_OK;
  JoinArgs j{g, {}, {}};
  for (int i = 0; i < (n > 1 ? n : 3); ++i) {
    const Mat& o = n > 1 ? qs[i].o[0] : q.o[i];
    j.o[i] = const_cast<void*>(o.p);
    j.ldo[i] = o.ld;
  }
  const int warps = g.sched.long_tiles * 2 * kEpiWarps * (is_plain(kEpi) ? kWarpCols : kFeat / 2) / kJoinCols;
  constexpr int per = join_threads(kEpi) / 32;
  cudaLaunchAttribute jat[2];
  cudaLaunchConfig_t join = launch_config(jat, (warps + per - 1) / per, 32 * per, 0, 1, &ctx);
  return cudaLaunchKernelEx(&join, k_ffn_join<kEpi, kF16>, j) == cudaSuccess ? MB_OK : MB_ERR_CUDA;
}

constexpr int kSkinnyPerSm = 3, kSkinnyStages = 3;
constexpr int kSkinnyMaxSmem = 227 * 1024;

template <int kEpi, bool kAMn, bool kF16>
int launch_skinny(const Product& q, Ctx& ctx) {
  // q is given as in the pair form (a: tokens, b: weights); the MMA swaps them
  auto kernel = &k_ffn_skinny<kEpi, kAMn, kF16>;
  static KernelEntry entry;
  int sms = 0;
  const int dev = current_device(&sms);
  if (dev < 0) return MB_ERR_CUDA;
  std::call_once(entry.once[dev], [&] {
    entry.rc[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSkinnyMaxSmem) ==
                            cudaSuccess
                        ? MB_OK
                        : MB_ERR_CUDA;
  });
  if (entry.rc[dev] != MB_OK) return entry.rc[dev];
  SkinnyArgs g{};
  g.tokens = (int)q.M;
  g.n = (int)((q.M + 15) / 16 * 16);
  g.rows = (int)q.N;
  constexpr int kPer = is_plain(kEpi) ? 128 : 64;
  const int64_t kb = (q.K + BK - 1) / BK, tiles = (q.N + kPer - 1) / kPer, KB = kb * q.nseg;
  if (KB > kMaxKb) return MB_ERR_TOO_LARGE;
  g.kb = (int)kb; g.nseg = q.nseg;
  const int stage = kTileA + g.n * BK * 2, partials = (int)q.M * kSkinnyPitch * 4;  // the ring's memory holds both
  g.tmem_cols = 32;
  while ((int)g.tmem_cols < g.n) g.tmem_cols *= 2;
  // As many CTAs on an SM as leave each kSkinnyStages stages. All that the memory lets
  // in must find TMEM columns too: CTAs of two clusters that waited for each other's
  // columns would never end.
  int per_sm = kSkinnyPerSm + 1, smem;
  do {
    --per_sm;
    smem = (228 / per_sm - 1) * 1024;
    g.st = (smem - 1024 - kBarBytes) / stage;
  } while (per_sm > 1 && (g.st < kSkinnyStages || g.st * stage < partials || per_sm * g.tmem_cols > 512));
  if (g.st < 1 || g.st * stage < partials || smem > kSkinnyMaxSmem) return MB_ERR_TOO_LARGE;
  // Split the contraction as far as all CTAs find room at once and keep four k-blocks
  // each.
  g.split = 1;
  while (g.split < 8 && tiles * 2 * g.split <= (int64_t)per_sm * sms && KB / (2 * g.split) >= 4) g.split *= 2;
  g.act = q.act;
  Maps m;
  bool ok = true;
  const int nw = is_plain(kEpi) ? q.nseg : 2;
  constexpr CUtensorMapDataType t16 = kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < nw; ++i)
    ok = ok && map_2d(&m.a[i], t16, q.b[i].p, q.b[i].rows, q.b[i].cols, q.b[i].ld, 64,
                      is_plain(kEpi) && !kAMn ? 128 : 64);
  for (int i = 0; i < q.nseg; ++i)
    ok = ok && map_2d(&m.b[i], t16, q.a[i].p, q.a[i].rows, q.a[i].cols, q.a[i].ld, 64, g.n);
  if (!ok) return MB_ERR_CUDA;
  for (int i = nw; i < 2; ++i) m.a[i] = m.a[0];  // every map the kernel prefetches is one
  for (int i = q.nseg; i < 2; ++i) m.b[i] = m.b[0];
  g.o0 = const_cast<void*>(q.o[0].p); g.ldo = q.o[0].ld;
  g.o1 = const_cast<void*>(q.o[1].p); g.ldu = q.o[1].ld;
  g.o2 = const_cast<void*>(q.o[2].p); g.ldh = q.o[2].ld;
  g.dh = q.dh.p; g.lddh = q.dh.ld;
  take_fault(kFaultFfn, &g.fault.unit, &g.fault.limit_ns);
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t cfg =
      launch_config(at, (int)(tiles * g.split), kSkinnyThreads, smem, g.split, &ctx);
  ctx.chained = cudaLaunchKernelEx(&cfg, kernel, m, g) == cudaSuccess;
  return ctx.chained ? MB_OK : MB_ERR_CUDA;
}

template <bool kF16>
int run_product(const Product& q, Ctx& ctx) {
  const bool skinny = q.M <= (is_plain(q.epi) ? kSkinnyTokensPlain : kSkinnyTokens);
  switch (q.epi) {
    case kGated:
      return skinny ? launch_skinny<kGated, false, kF16>(q, ctx) : launch_pair<kGated, false, false, kF16>(&q, 1, ctx);
    case kGatedBwd:
      return skinny ? launch_skinny<kGatedBwd, false, kF16>(q, ctx)
                    : launch_pair<kGatedBwd, false, false, kF16>(&q, 1, ctx);
    case kGatedBwdF32:
      return skinny ? launch_skinny<kGatedBwdF32, false, kF16>(q, ctx)
                    : launch_pair<kGatedBwdF32, false, false, kF16>(&q, 1, ctx);
    case kPlainF32:
      return skinny ? launch_skinny<kPlainF32, true, kF16>(q, ctx)
                    : launch_pair<kPlainF32, false, true, kF16>(&q, 1, ctx);
    default:
      if (q.b_mn)
        return skinny ? launch_skinny<kPlain, true, kF16>(q, ctx) : launch_pair<kPlain, true, true, kF16>(&q, 1, ctx);
      return skinny ? launch_skinny<kPlain, false, kF16>(q, ctx) : launch_pair<kPlain, false, false, kF16>(&q, 1, ctx);
  }
}

int product(int dtype, const Product& q, Ctx& ctx) {
  return dtype == MB_F16 ? run_product<true>(q, ctx) : run_product<false>(q, ctx);
}

// Products over 16-bit B stored [K, N], in one launch.
int products(int dtype, const Product* q, int n, Ctx& ctx) {
  if (n == 0) return MB_OK;
  return dtype == MB_F16 ? launch_pair<kPlain, true, true, true>(q, n, ctx)
                         : launch_pair<kPlain, true, true, false>(q, n, ctx);
}

// The call's context over the joining part of its workspace (its first kJoinBytes).
Ctx make_ctx(void* workspace, cudaStream_t stream) { return {stream, static_cast<float*>(workspace), false}; }

constexpr int64_t kMaxDim = (int64_t)1 << 30;

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
size_t area(int64_t rows, int64_t cols) { return ((size_t)rows * (size_t)pad8(cols) * 2 + 255) / 256 * 256; }

// A caller's matrix: whole elements, rows that do not overlap.
int check_mat(const void* p, int64_t cols, int64_t ld) {
  if (!p || ld < cols) return MB_ERR_ARG;
  if (!aligned(p, 2) || ld >= ((int64_t)1 << 36)) return MB_ERR_ALIGN;
  return MB_OK;
}

// The end of a call's workspace, from which padded copies of unaligned matrices are cut.
class Padding {
 public:
  Padding(void* base, size_t bytes) : next_(static_cast<uint8_t*>(base)), left_(bytes) {}

  // The matrix as the kernels may read it.
  Mat in(const void* p, int64_t rows, int64_t cols, int64_t ld) {
    if (!p) return {};
    return fits(p, rows, ld) ? Mat{p, rows, cols, rows > 1 ? ld : pad8(cols)} : copy(in_, n_in_, p, rows, cols, ld, false);
  }
  // The matrix as the kernels may write it.
  Mat out(void* p, int64_t rows, int64_t cols, int64_t ld) {
    if (!p) return {};
    return fits(p, rows, ld) ? Mat{p, rows, cols, rows > 1 ? ld : pad8(cols)} : copy(out_, n_out_, p, rows, cols, ld, true);
  }
  int status() const { return rc_; }
  int before(cudaStream_t st) const { return launch(in_, n_in_, st); }
  int after(cudaStream_t st) const { return launch(out_, n_out_, st); }

 private:
  static bool fits(const void* p, int64_t rows, int64_t ld) { return aligned(p, 16) && (ld % 8 == 0 || rows <= 1); }

  Mat copy(CopyJobs& jobs, int& n, const void* p, int64_t rows, int64_t cols, int64_t ld, bool back) {
    const size_t need = area(rows, cols);
    if (n == kMaxCopies || left_ < need) {
      rc_ = MB_ERR_ALIGN;
      return {};
    }
    const Mat m{next_, rows, cols, pad8(cols)};
    next_ += need;
    left_ -= need;
    uint16_t *mine = static_cast<uint16_t*>(const_cast<void*>(m.p)), *theirs = static_cast<uint16_t*>(const_cast<void*>(p));
    jobs.j[n++] = back ? CopyJob{mine, theirs, m.ld, ld, rows, cols} : CopyJob{theirs, mine, ld, m.ld, rows, cols};
    return m;
  }
  static int launch(const CopyJobs& jobs, int n, cudaStream_t st) {
    if (n == 0) return MB_OK;
    int64_t rows = 0;
    for (int i = 0; i < n; ++i) rows = jobs.j[i].rows > rows ? jobs.j[i].rows : rows;
    const int64_t blocks = (rows + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
    k_ffn_copy<<<dim3((unsigned)(blocks < 1184 ? blocks : 1184), (unsigned)n), kCopyThreads, 0, st>>>(jobs);
    return cudaGetLastError() == cudaSuccess ? MB_OK : MB_ERR_CUDA;
  }

  uint8_t* next_;
  size_t left_;
  CopyJobs in_, out_;
  int n_in_ = 0, n_out_ = 0, rc_ = MB_OK;
};

int check_args(const mb_ffn_args* a, bool need_x, bool need_down) {
  if (!a) return MB_ERR_ARG;
  if (a->dtype != MB_BF16 && a->dtype != MB_F16) return MB_ERR_ARG;
  if (a->activation != MB_ACT_SILU && a->activation != MB_ACT_GELU_TANH) return MB_ERR_ARG;
  if (a->tokens < 0 || a->d <= 0 || a->f <= 0) return MB_ERR_ARG;
  if (a->tokens > kMaxDim || a->d > kMaxDim || a->f > kMaxDim) return MB_ERR_TOO_LARGE;
  int rc = MB_OK;
  if (need_x && a->tokens > 0) rc = check_mat(a->x, a->d, a->ldx);
  if (rc == MB_OK) rc = check_mat(a->gate, a->d, a->ld_gate);
  if (rc == MB_OK) rc = check_mat(a->up, a->d, a->ld_up);
  if (rc == MB_OK && need_down) rc = check_mat(a->down, a->f, a->ld_down);
  return rc;
}

// A call's contractions, in k-blocks, are checked before its first launch: one that is
// refused has written nothing.
bool too_long(int64_t k, int nseg = 1) { return (k + BK - 1) / BK * nseg > kMaxKb; }

Product gated_product(const mb_ffn_args* a, const Mat& x, const Mat& gate, const Mat& up) {
  Product q;
  q.epi = kGated;
  q.a[0] = x;
  q.b[0] = gate;
  q.b[1] = up;
  q.M = a->tokens; q.N = a->f; q.K = a->d;
  q.act = a->activation;
  return q;
}

int zero_rows(void* p, int64_t rows, int64_t cols, int64_t ld, cudaStream_t st) {
  return cudaMemset2DAsync(p, (size_t)ld * 2, 0, (size_t)cols * 2, (size_t)rows, st) == cudaSuccess ? MB_OK : MB_ERR_CUDA;
}

}  // namespace ffn
}  // namespace mb

using namespace mb;
using namespace mb::ffn;

extern "C" {

MB_API size_t mb_ffn_padding_bytes(int64_t tokens, int64_t d, int64_t f) {
  if (tokens <= 0 || d <= 0 || f <= 0 || tokens > kMaxDim || d > kMaxDim || f > kMaxDim) return 0;
  // x, dy, dx or y over d; dh or h over f; the weights and their gradients
  return 3 * area(tokens, d) + area(tokens, f) + 4 * area(f, d) + 2 * area(d, f);
}

MB_API size_t mb_gated_linear_workspace_bytes(int64_t tokens) {
  return tokens <= 0 || tokens > kMaxDim ? 0 : join_bytes(tokens);
}

MB_API size_t mb_feed_forward_workspace_bytes(int64_t tokens, int64_t f) {
  if (tokens <= 0 || f <= 0 || tokens > kMaxDim || f > kMaxDim) return 0;
  return join_bytes(tokens) + area(tokens, f);
}

// Both forward entries: without down, y is h.
static int forward(const mb_ffn_args* a, bool with_down, void* y, int64_t ldy, void* workspace, size_t workspace_bytes,
                   cudaStream_t st) {
  int rc = check_args(a, true, with_down);
  if (rc != MB_OK) return rc;
  const int64_t T = a->tokens, d = a->d, f = a->f, width = with_down ? d : f;
  if (T == 0) return MB_OK;
  if (too_long(d) || (with_down && too_long(f))) return MB_ERR_TOO_LARGE;
  rc = check_mat(y, width, ldy);
  if (rc != MB_OK) return rc;
  const size_t need = with_down ? mb_feed_forward_workspace_bytes(T, f) : mb_gated_linear_workspace_bytes(T);
  if ((need > 0 && !workspace) || workspace_bytes < need) return MB_ERR_ARG;
  if (!aligned(workspace, 256)) return MB_ERR_ALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Padding pad(ws + need, workspace ? workspace_bytes - need : 0);
  const Mat x = pad.in(a->x, T, d, a->ldx), gate = pad.in(a->gate, f, d, a->ld_gate), up = pad.in(a->up, f, d, a->ld_up);
  const Mat down = with_down ? pad.in(a->down, d, f, a->ld_down) : Mat{}, out = pad.out(y, T, width, ldy);
  if (pad.status() != MB_OK) return pad.status();
  rc = pad.before(st);
  if (rc != MB_OK) return rc;
  Ctx ctx = make_ctx(workspace, st);  // its first kernel is not chained to the copies: it reads them at once
  Product q = gated_product(a, x, gate, up);
  q.o[0] = with_down ? Mat{ws + join_bytes(T), T, f, pad8(f)} : out;
  rc = product(a->dtype, q, ctx);
  if (rc == MB_OK && with_down) {
    Product p;
    p.a[0] = q.o[0];
    p.b[0] = down;
    p.o[0] = out;
    p.M = T; p.N = d; p.K = f;
    rc = product(a->dtype, p, ctx);
  }
  return rc == MB_OK ? pad.after(st) : rc;
}

MB_API int mb_gated_linear(const mb_ffn_args* a, void* h, int64_t ldh, void* workspace, size_t workspace_bytes,
                           mb_stream_t stream) {
  return forward(a, false, h, ldh, workspace, workspace_bytes, (cudaStream_t)stream);
}

MB_API int mb_feed_forward(const mb_ffn_args* a, void* y, int64_t ldy, void* workspace, size_t workspace_bytes,
                           mb_stream_t stream) {
  return forward(a, true, y, ldy, workspace, workspace_bytes, (cudaStream_t)stream);
}

MB_API size_t mb_feed_forward_backward_workspace_bytes(int64_t tokens, int64_t d, int64_t f, int32_t from_codes,
                                                       int32_t with_down) {
  if (tokens <= 0 || d <= 0 || f <= 0 || tokens > kMaxDim || d > kMaxDim || f > kMaxDim) return 0;
  // the weight gradients always run on pairs; dg, du; with down: h and an FP32 dh
  return kJoinBytes + (with_down ? 5 : 2) * area(tokens, f) + (from_codes ? area(tokens, d) : 0);
}

MB_API int mb_feed_forward_backward(const mb_ffn_args* a, const mb_ffn_grads* r, void* workspace,
                                    size_t workspace_bytes, mb_stream_t stream) {
  if (!a || !r) return MB_ERR_ARG;
  const bool from_codes = r->codes != nullptr, with_down = a->down != nullptr;
  int rc = check_args(a, !from_codes, with_down);
  if (rc != MB_OK) return rc;
  const int64_t T = a->tokens, d = a->d, f = a->f;
  if (r->dx && T > 0) rc = check_mat(r->dx, d, r->lddx);
  if (rc == MB_OK && r->dgate) rc = check_mat(r->dgate, d, r->ld_dgate);
  if (rc == MB_OK && r->dup) rc = check_mat(r->dup, d, r->ld_dup);
  if (rc == MB_OK && r->ddown) rc = with_down ? check_mat(r->ddown, f, r->ld_ddown) : MB_ERR_ARG;
  if (rc != MB_OK) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (T == 0) {  // sums over no tokens
    if (r->dgate) rc = zero_rows(r->dgate, f, d, r->ld_dgate, st);
    if (rc == MB_OK && r->dup) rc = zero_rows(r->dup, f, d, r->ld_dup, st);
    if (rc == MB_OK && r->ddown) rc = zero_rows(r->ddown, d, f, r->ld_ddown, st);
    return rc;
  }
  if (!r->dx && !r->dgate && !r->dup && !r->ddown) return MB_OK;
  if (too_long(d) || (r->dx && too_long(f, 2)) || ((r->dgate || r->dup || r->ddown) && too_long(T))) return MB_ERR_TOO_LARGE;
  rc = check_mat(r->dy, with_down ? d : f, r->lddy);
  if (rc != MB_OK) return rc;
  if (from_codes && !r->scales) return MB_ERR_ARG;
  const size_t need = mb_feed_forward_backward_workspace_bytes(T, d, f, from_codes ? 1 : 0, with_down ? 1 : 0);
  if (!workspace || workspace_bytes < need) return MB_ERR_ARG;
  if (!aligned(workspace, 256)) return MB_ERR_ALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Padding pad(ws + need, workspace_bytes - need);
  ws += kJoinBytes;
  const int64_t fp = pad8(f);
  const Mat dg{ws, T, f, fp}, du{ws + area(T, f), T, f, fp};
  ws += 2 * area(T, f);
  const Mat dy = pad.in(r->dy, T, with_down ? d : f, r->lddy);
  Mat dh = dy, h;
  if (with_down) {
    h = {ws, T, f, fp};
    dh = {ws + area(T, f), T, f, fp};
    ws += 3 * area(T, f);
  }
  const Mat x = from_codes ? Mat{ws, T, d, pad8(d)} : pad.in(a->x, T, d, a->ldx);
  const Mat gate = pad.in(a->gate, f, d, a->ld_gate), up = pad.in(a->up, f, d, a->ld_up);
  const Mat down = with_down ? pad.in(a->down, d, f, a->ld_down) : Mat{};
  const Mat dx = pad.out(r->dx, T, d, r->lddx), dgate = pad.out(r->dgate, f, d, r->ld_dgate);
  const Mat dup = pad.out(r->dup, f, d, r->ld_dup), ddown = pad.out(r->ddown, d, f, r->ld_ddown);
  if (pad.status() != MB_OK) return pad.status();
  rc = pad.before(st);
  if (rc != MB_OK) return rc;
  if (from_codes) {
    rc = act_unpack(r->codes, r->scales, T, d, const_cast<void*>(x.p), a->dtype, pad8(d), st);
    if (rc != MB_OK) return rc;
  }
  Ctx ctx = make_ctx(workspace, st);
  if (with_down) {
    Product q;
    q.epi = kPlainF32;
    q.a[0] = dy;
    q.b[0] = down;
    q.b_mn = true;
    q.o[0] = dh;
    q.M = T; q.N = f; q.K = d;
    rc = product(a->dtype, q, ctx);
    if (rc != MB_OK) return rc;
  }
  {
    Product q = gated_product(a, x, gate, up);
    q.epi = with_down ? kGatedBwdF32 : kGatedBwd;
    q.dh = dh;
    q.o[0] = dg; q.o[1] = du;
    if (r->ddown) q.o[2] = h;
    rc = product(a->dtype, q, ctx);
    if (rc != MB_OK) return rc;
  }
  // dx and the weight gradients need each other's results for nothing: one launch, by
  // falling contraction (a few tokens' dx is a stream over the weights, for the skinny
  // kernel)
  Product grads[kMaxProblems];
  int n = 0;
  Product q;
  if (r->dx) {
    q.nseg = 2;
    q.a[0] = dg; q.a[1] = du;
    q.b[0] = gate; q.b[1] = up;
    q.b_mn = true;
    q.o[0] = dx;
    q.M = T; q.N = d; q.K = f;
    if (T <= kSkinnyTokensPlain) {
      rc = product(a->dtype, q, ctx);
      if (rc != MB_OK) return rc;
    }
  }
  const bool dx_here = r->dx && T > kSkinnyTokensPlain, dx_last = q.kblocks() < (T + BK - 1) / BK;
  if (dx_here && !dx_last) grads[n++] = q;
  auto weight = [&](const Mat& left, const Mat& right, const Mat& out) {  // out = left^T right
    if (!out.p) return;
    Product& q = grads[n++];
    q.a_mn = q.b_mn = true;
    q.a[0] = left;
    q.b[0] = right;
    q.o[0] = out;
    q.M = left.cols; q.N = right.cols; q.K = T;
  };
  weight(dg, x, dgate);
  weight(du, x, dup);
  weight(dy, h, ddown);
  if (dx_here && dx_last) grads[n++] = q;
  rc = products(a->dtype, grads, n, ctx);
  return rc == MB_OK ? pad.after(st) : rc;
}

MB_API int mb_ffn_status(void) {
  int32_t err = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return MB_ERR_CUDA;
  if (cudaMemcpyFromSymbol(&err, g_ffn_err, sizeof(err)) != cudaSuccess) return MB_ERR_CUDA;
  if (err == 0) return MB_OK;
  err = 0;
  if (cudaMemcpyToSymbol(g_ffn_err, &err, sizeof(err)) != cudaSuccess) return MB_ERR_CUDA;
  return MB_ERR_TIMEOUT;
}

}  // extern "C"
