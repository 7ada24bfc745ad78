// Activation checkpoints in 8 bits: save (pack) and restore (unpack).
//
// A stage boundary x [rows, d] (FP32, FP16 or BF16; d contiguous, any row
// stride) is kept as one E4M3FN code per element and one power-of-two scale per
// 128 features of a row (uint8 exponent + 127):
//   a = max |finite x_j| of the block = m 2^e, 1 <= m < 2
//   s = e - 8 if m <= 1.75 else e - 7, at least -127; 0 for a zero block
//   code_j = E4M3(x_j 2^-s), round to nearest even; a nonfinite x_j becomes the
//   NaN code, and its neighbours keep theirs
//   value  = code_j 2^s
// so the largest magnitude lands in (224, 448]. Both scalings are exact: the one
// rounding is the code's (relative 2^-4 of a normal code's value). A code has 4
// significant bits, so a power-of-two scale makes the restored value exact in
// BF16 and, inside its range, in FP16: the tensor cores of the backward pass
// read exactly what the checkpoint holds. Values that round past the output
// type's range restore as its largest finite value.
//
// Both directions are bound by HBM: in + 1 + 1/128 bytes per element (and the
// same back). 16 lanes own one 128-feature block, 8 elements each (one 16- or
// 32-byte load of x, one 8-byte store of codes), and a half-warp has several blocks' loads in flight
// before any arithmetic. The block maximum is an integer maximum over the magnitude
// bits (two 16-bit values at a time), which also shows infinities and NaN. A matrix
// without gaps whose rows are whole blocks is walked as one row (no division).
#include <cuda_fp8.h>

#include "mb_common.cuh"

namespace mb {
namespace {

constexpr int kBlk = 128;     // features per scale
constexpr int kLaneElems = 8; // 16 lanes x 8 = one block
constexpr int kUnroll = 2;  // blocks a half-warp has in flight: 4 cost 15 % at 8191 x 1000, 1 up to 12 %

// How a launch walks its matrix: any alignment and size; rows whose 8-element
// groups are aligned and fit 32-bit block indexes; the same as one long row.
enum Mode { kAny = 0, kRows = 1, kFlat = 2 };

struct Shape {
  int64_t rows, d, ld;  // ld: row pitch of the 16/32-bit side, in elements
  int64_t blocks;       // scale blocks per row
};

// A lane's 8 elements as they lie in memory: 4 or 8 words.
template <int DT> constexpr int kWords = DT == MB_F32 ? 8 : 4;

template <int DT>
__device__ __forceinline__ void load_raw(const void* p, int64_t e, uint32_t (&w)[kWords<DT>]) {
  const uint8_t* q = static_cast<const uint8_t*>(p) + e * (DT == MB_F32 ? 4 : 2);
  if constexpr (DT == MB_F32) {
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(q));
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(q));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
}

template <int DT>
__device__ __forceinline__ void load_raw_any(const void* p, int64_t e, int n, uint32_t (&w)[kWords<DT>]) {
#pragma unroll
  for (int i = 0; i < kWords<DT>; ++i) w[i] = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= n) continue;
    if constexpr (DT == MB_F32) w[j] = static_cast<const uint32_t*>(p)[e + j];
    else w[j / 2] |= (uint32_t)static_cast<const uint16_t*>(p)[e + j] << (16 * (j & 1));
  }
}

template <int DT>
__device__ __forceinline__ float raw_value(const uint32_t (&w)[kWords<DT>], int j) {
  if constexpr (DT == MB_F32) return __uint_as_float(w[j]);
  if constexpr (DT == MB_BF16) return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  if constexpr (DT == MB_F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j / 2]));
    return j & 1 ? f.y : f.x;
  }
}

// Largest magnitude of the block's 128 elements, as FP32 bits; the infinity's bits or
// more when one of them is not finite. All 16 lanes get it.
template <int DT>
__device__ __forceinline__ uint32_t block_top(const uint32_t (&w)[kWords<DT>], uint32_t half) {
  if constexpr (DT == MB_F32) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, w[i] & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(half, top, o));
    return top;
  } else {
    uint32_t two = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) two = __vmaxu2(two, w[i] & 0x7fff7fffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) two = __vmaxu2(two, __shfl_xor_sync(half, two, o));
    const uint32_t top = max(two & 0xffffu, two >> 16);
    if constexpr (DT == MB_BF16) return top << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
  }
}

// Elements of a row that lane group `l16` of block `blk` owns (0..8).
__device__ __forceinline__ int owned(const Shape& s, int64_t blk, int l16) {
  const int64_t left = s.d - (blk * kBlk + l16 * kLaneElems);
  return left >= kLaneElems ? kLaneElems : left > 0 ? (int)left : 0;
}

template <int MODE> struct Index {
  using T = uint32_t;
};
template <> struct Index<kAny> {
  using T = int64_t;
};

// Where block b's part of this lane lies.
template <int MODE>
struct Place {
  int64_t wide, code;  // element offsets of x / out and of codes
  int n;               // elements owned
  __device__ __forceinline__ Place(const Shape& s, typename Index<MODE>::T b, typename Index<MODE>::T total, int l16) {
    wide = code = 0;
    n = 0;
    if (b >= total) return;
    if constexpr (MODE == kFlat) {
      wide = code = (int64_t)b * kBlk + l16 * kLaneElems;
      n = 8;
    } else {
      const typename Index<MODE>::T nb = (typename Index<MODE>::T)s.blocks, row = b / nb, blk = b - row * nb;
      const int64_t in = (int64_t)blk * kBlk + l16 * kLaneElems;
      wide = (int64_t)row * s.ld + in;
      code = (int64_t)row * s.d + in;
      n = owned(s, blk, l16);
    }
  }
};

template <int DT, int MODE>
__global__ void __launch_bounds__(kThreads) k_act_pack(const void* __restrict__ x, Shape s,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  using Idx = typename Index<MODE>::T;
  const int l16 = threadIdx.x & 15;
  const Idx total = (Idx)(s.rows * s.blocks);
  const Idx step = (Idx)gridDim.x * (kThreads / 16);
  // the 16 lanes of a half-warp share every block index, so they run (or leave)
  // together and the shuffles name exactly those lanes
  const uint32_t half = (threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu;
  for (Idx b0 = (Idx)blockIdx.x * (kThreads / 16) + threadIdx.x / 16; b0 < total; b0 += step * kUnroll) {
    uint32_t w[kUnroll][kWords<DT>];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Place<MODE> at(s, b0 + (Idx)u * step, total, l16);
      if constexpr (MODE == kAny) {
        load_raw_any<DT>(x, at.wide, at.n, w[u]);
      } else {
#pragma unroll
        for (int i = 0; i < kWords<DT>; ++i) w[u][i] = 0;
        if (at.n) load_raw<DT>(x, at.wide, w[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Idx b = b0 + (Idx)u * step;
      if (b >= total) break;
      const Place<MODE> at(s, b, total, l16);
      uint32_t top = block_top<DT>(w[u], half);
      const bool bad = top >= 0x7f800000u;
      if (bad) {  // the maximum of the finite magnitudes
        top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t m = __float_as_uint(raw_value<DT>(w[u], j)) & 0x7fffffffu;
          if (m < 0x7f800000u) top = max(top, m);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(half, top, o));
      }
      // biased scale exponent (s + 127): e - 8 + 127 = field - 8, one more when
      // the mantissa passes 1.75; a subnormal maximum (field 0) lands on the floor
      int se = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
      se = top == 0 ? 127 : se < 0 ? 0 : se;
      const float inv = __uint_as_float((uint32_t)(254 - se) << 23);  // 2^-s; se <= 247, so always normal
      uint32_t pk[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = __fmul_rn(raw_value<DT>(w[u], 4 * h + j), inv);
        if (bad) {  // a NaN, not the largest code
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!is_finite(raw_value<DT>(w[u], 4 * h + j))) q[j] = __int_as_float(0x7fc00000);
        }
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
        pk[h] = lo | (hi << 16);
      }
      uint8_t* dst = codes + at.code;
      if constexpr (MODE == kAny) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < at.n) dst[j] = (uint8_t)(pk[j >> 2] >> (8 * (j & 3)));
      } else {
        if (at.n) *reinterpret_cast<uint2*>(dst) = make_uint2(pk[0], pk[1]);
      }
      if (l16 == 0) scales[b] = (uint8_t)se;
    }
  }
}

template <int DT, int MODE>
__global__ void __launch_bounds__(kThreads) k_act_unpack(const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, Shape s, void* out) {
  using Idx = typename Index<MODE>::T;
  const int l16 = threadIdx.x & 15;
  const Idx total = (Idx)(s.rows * s.blocks);
  const Idx step = (Idx)gridDim.x * (kThreads / 16);
  // the largest finite value of the output, and the smallest scale exponent
  // (biased) whose 448 2^s passes it
  constexpr float kTop = DT == MB_F16 ? 65504.0f : DT == MB_BF16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  constexpr int kClampFrom = DT == MB_F16 ? 127 + 8 : 127 + 120;
  for (Idx b0 = (Idx)blockIdx.x * (kThreads / 16) + threadIdx.x / 16; b0 < total; b0 += step * kUnroll) {
    uint2 c[kUnroll];
    int se[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Idx b = b0 + (Idx)u * step;
      const Place<MODE> at(s, b, total, l16);
      c[u] = make_uint2(0, 0);
      se[u] = 127;
      if (b < total) se[u] = scales[b];
      if constexpr (MODE == kAny) {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < at.n) w[j >> 2] |= (uint32_t)codes[at.code + j] << (8 * (j & 3));
        c[u] = make_uint2(w[0], w[1]);
      } else {
        if (at.n) c[u] = __ldcs(reinterpret_cast<const uint2*>(codes + at.code));
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Place<MODE> at(s, b0 + (Idx)u * step, total, l16);
      if (at.n == 0) continue;
      // 2^s; the smallest exponent's scale (2^-127) is a subnormal float
      const float scale = __uint_as_float(se[u] > 0 ? (uint32_t)se[u] << 23 : 0x400000u);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_fp8x2_storage_t two = (__nv_fp8x2_storage_t)((i < 2 ? c[u].x : c[u].y) >> (16 * (i & 1)));
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[2 * i] = __fmul_rn(f.x, scale);
        v[2 * i + 1] = __fmul_rn(f.y, scale);
      }
      if (se[u] >= kClampFrom) {
#pragma unroll
        for (int j = 0; j < 8; ++j)  // NaN compares false and stays
          v[j] = v[j] > kTop ? kTop : v[j] < -kTop ? -kTop : v[j];
      }
      if constexpr (MODE == kAny) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < at.n) store1<DT>(out, at.wide + j, v[j]);
      } else if constexpr (DT == MB_F32) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                         static_cast<float*>(out) + at.wide),
                     "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
      } else {
        uint32_t pk[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (DT == MB_BF16) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            pk[i] = *reinterpret_cast<const uint32_t*>(&t);
          } else {
            const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            pk[i] = *reinterpret_cast<const uint32_t*>(&t);
          }
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at.wide) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
      }
    }
  }
}

// Rows and row lengths this file's index arithmetic covers: element offsets and
// block counts fit 62 bits.
bool shape_ok(int64_t rows, int64_t d, int64_t ld) {
  return rows >= 0 && d > 0 && ld >= d && ld <= ((int64_t)1 << 40) && rows <= ((int64_t)1 << 62) / ld;
}

// The mode of a launch; a flat one's shape becomes one row. Block indexes stay below
// 2^30 in 32-bit modes, so that the loop's overshoot cannot wrap.
int pick_mode(Shape& s, const void* wide, int elem, const void* codes) {
  s.blocks = (s.d + kBlk - 1) / kBlk;
  if (!aligned(wide, 8 * elem) || (s.ld * elem) % (8 * elem) || !aligned(codes, 8) || s.d % 8 ||
      s.rows * s.blocks >= ((int64_t)1 << 30))
    return kAny;
  if (s.d % kBlk || s.ld != s.d) return kRows;
  s = {1, s.rows * s.d, s.rows * s.d, s.rows * s.blocks};
  return kFlat;
}

template <int DT, int MODE>
int launch_pack(const void* x, const Shape& s, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  const int64_t per_cta = (int64_t)(kThreads / 16) * kUnroll;
  const int grid = grid_for(reinterpret_cast<const void*>(&k_act_pack<DT, MODE>), (s.rows * s.blocks + per_cta - 1) / per_cta);
  k_act_pack<DT, MODE><<<grid, kThreads, 0, st>>>(x, s, codes, scales);
  return cudaGetLastError() == cudaSuccess ? MB_OK : MB_ERR_CUDA;
}

template <int DT>
int pack(const void* x, Shape s, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  switch (pick_mode(s, x, DT == MB_F32 ? 4 : 2, codes)) {
    case kFlat: return launch_pack<DT, kFlat>(x, s, codes, scales, st);
    case kRows: return launch_pack<DT, kRows>(x, s, codes, scales, st);
    default: return launch_pack<DT, kAny>(x, s, codes, scales, st);
  }
}

template <int DT, int MODE>
int launch_unpack(const uint8_t* codes, const uint8_t* scales, const Shape& s, void* out, cudaStream_t st) {
  const int64_t per_cta = (int64_t)(kThreads / 16) * kUnroll;
  const int grid =
      grid_for(reinterpret_cast<const void*>(&k_act_unpack<DT, MODE>), (s.rows * s.blocks + per_cta - 1) / per_cta);
  k_act_unpack<DT, MODE><<<grid, kThreads, 0, st>>>(codes, scales, s, out);
  return cudaGetLastError() == cudaSuccess ? MB_OK : MB_ERR_CUDA;
}

template <int DT>
int unpack(const uint8_t* codes, const uint8_t* scales, Shape s, void* out, cudaStream_t st) {
  switch (pick_mode(s, out, DT == MB_F32 ? 4 : 2, codes)) {
    case kFlat: return launch_unpack<DT, kFlat>(codes, scales, s, out, st);
    case kRows: return launch_unpack<DT, kRows>(codes, scales, s, out, st);
    default: return launch_unpack<DT, kAny>(codes, scales, s, out, st);
  }
}

}  // namespace

int act_unpack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t d, void* out, int out_dtype,
               int64_t ld, cudaStream_t st) {
  if (!shape_ok(rows, d, ld)) return MB_ERR_ARG;
  if (rows == 0) return MB_OK;
  if (!codes || !scales || !out) return MB_ERR_ARG;
  const Shape s{rows, d, ld, 0};
  switch (out_dtype) {
    case MB_F32: return unpack<MB_F32>(codes, scales, s, out, st);
    case MB_F16: return unpack<MB_F16>(codes, scales, s, out, st);
    case MB_BF16: return unpack<MB_BF16>(codes, scales, s, out, st);
    default: return MB_ERR_ARG;
  }
}

}  // namespace mb

using namespace mb;

extern "C" {

MB_API int mb_act_pack(const void* x, int32_t dtype, int64_t rows, int64_t d, int64_t ld, uint8_t* codes,
                       uint8_t* scales, mb_stream_t stream) {
  if (!shape_ok(rows, d, ld)) return MB_ERR_ARG;
  if (dtype != MB_F32 && dtype != MB_F16 && dtype != MB_BF16) return MB_ERR_ARG;
  if (rows == 0) return MB_OK;
  if (!x || !codes || !scales) return MB_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const Shape s{rows, d, ld, 0};
  if (dtype == MB_F32) return pack<MB_F32>(x, s, codes, scales, st);
  if (dtype == MB_F16) return pack<MB_F16>(x, s, codes, scales, st);
  return pack<MB_BF16>(x, s, codes, scales, st);
}

MB_API int mb_act_unpack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t d, void* out,
                         int32_t out_dtype, int64_t ld, mb_stream_t stream) {
  return act_unpack(codes, scales, rows, d, out, out_dtype, ld, (cudaStream_t)stream);
}

}  // extern "C"
