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
// same back). 16 lanes own one 128-feature block, 8 elements each (one 16-byte
// load of a 16-bit type, one 8-byte store of codes), and every half-warp has
// kUnroll blocks' loads in flight before any arithmetic.
#include <cuda_fp8.h>

#include "mb_common.cuh"

namespace mb {
namespace {

constexpr int kBlk = 128;     // features per scale
constexpr int kLaneElems = 8; // 16 lanes x 8 = one block
constexpr int kUnroll = 4;

struct Shape {
  int64_t rows, d, ld;  // ld: row pitch of the 16/32-bit side, in elements
  int64_t blocks;       // scale blocks per row
  int vec;              // every full block's lane group is 16-byte (codes: 8-byte) aligned
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t e, int n, bool vec, float (&v)[8]) {
  if (vec && n == 8) {
    if constexpr (DT == MB_F32) {
      const float4 a = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(p) + e));
      const float4 b = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(p) + e) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 q = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + e));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == MB_BF16) {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? load1<DT>(p, e + j) : 0.0f;
  }
}

// Elements of a row that lane group `l16` of block `blk` owns (0..8).
__device__ __forceinline__ int owned(const Shape& s, int64_t blk, int l16) {
  const int64_t left = s.d - (blk * kBlk + l16 * kLaneElems);
  return left >= kLaneElems ? kLaneElems : left > 0 ? (int)left : 0;
}

template <int DT, typename Idx>
__global__ void __launch_bounds__(kThreads) k_act_pack(const void* __restrict__ x, Shape s,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int l16 = threadIdx.x & 15;
  const Idx total = (Idx)(s.rows * s.blocks);
  const Idx step = (Idx)gridDim.x * (kThreads / 16);
  const Idx nb = (Idx)s.blocks;
  // the 16 lanes of a half-warp share every block index, so they run (or leave)
  // together and the shuffles below name exactly those lanes
  const uint32_t half = (threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu;
  for (Idx b0 = (Idx)blockIdx.x * (kThreads / 16) + threadIdx.x / 16; b0 < total; b0 += step * kUnroll) {
    float v[kUnroll][8];
    Idx row[kUnroll], blk[kUnroll];
    int n[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Idx b = b0 + (Idx)u * step;
      n[u] = 0;
      row[u] = blk[u] = 0;
      if (b < total) {
        row[u] = b / nb;
        blk[u] = b - row[u] * nb;
        n[u] = owned(s, blk[u], l16);
      }
      load8<DT>(x, (int64_t)row[u] * s.ld + (int64_t)blk[u] * kBlk + l16 * kLaneElems, n[u], s.vec != 0, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Idx b = b0 + (Idx)u * step;
      if (b >= total) break;
      // magnitudes compare as integers; infinities and NaN come out on top
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[u][j]) & 0x7fffffffu);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(half, top, o));
      const bool bad = top >= 0x7f800000u;
      if (bad) {  // the maximum of the finite magnitudes
        top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t m = __float_as_uint(v[u][j]) & 0x7fffffffu;
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
        for (int j = 0; j < 4; ++j) {
          const float t = v[u][4 * h + j];
          q[j] = bad && !is_finite(t) ? __int_as_float(0x7fc00000) : __fmul_rn(t, inv);
        }
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
        pk[h] = lo | (hi << 16);
      }
      uint8_t* dst = codes + (int64_t)row[u] * s.d + (int64_t)blk[u] * kBlk + l16 * kLaneElems;
      if (s.vec && n[u] == 8) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pk[0], pk[1]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n[u]) dst[j] = (uint8_t)(pk[j >> 2] >> (8 * (j & 3)));
      }
      if (l16 == 0) scales[b] = (uint8_t)se;
    }
  }
}

template <int DT, typename Idx>
__global__ void __launch_bounds__(kThreads) k_act_unpack(const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, Shape s, void* out) {
  const int l16 = threadIdx.x & 15;
  const Idx total = (Idx)(s.rows * s.blocks);
  const Idx step = (Idx)gridDim.x * (kThreads / 16);
  const Idx nb = (Idx)s.blocks;
  // the largest finite value of the output, and the smallest scale exponent
  // (biased) whose 448 2^s passes it
  constexpr float kTop = DT == MB_F16 ? 65504.0f : DT == MB_BF16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  constexpr int kClampFrom = DT == MB_F16 ? 127 + 8 : 127 + 120;
  for (Idx b0 = (Idx)blockIdx.x * (kThreads / 16) + threadIdx.x / 16; b0 < total; b0 += step * kUnroll) {
    uint2 c[kUnroll];
    int se[kUnroll], n[kUnroll];
    Idx row[kUnroll], blk[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Idx b = b0 + (Idx)u * step;
      n[u] = 0;
      row[u] = blk[u] = 0;
      se[u] = 127;
      c[u] = make_uint2(0, 0);
      if (b >= total) continue;
      row[u] = b / nb;
      blk[u] = b - row[u] * nb;
      n[u] = owned(s, blk[u], l16);
      se[u] = scales[b];
      const uint8_t* src = codes + (int64_t)row[u] * s.d + (int64_t)blk[u] * kBlk + l16 * kLaneElems;
      if (s.vec && n[u] == 8) {
        c[u] = __ldcs(reinterpret_cast<const uint2*>(src));
      } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n[u]) w[j >> 2] |= (uint32_t)src[j] << (8 * (j & 3));
        c[u] = make_uint2(w[0], w[1]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (n[u] == 0) continue;
      // 2^s; the two smallest exponents' scales (0: 2^-127) are subnormal floats
      const float scale = __uint_as_float(se[u] > 0 ? (uint32_t)se[u] << 23 : 0x400000u);
      const uint32_t w[2] = {c[u].x, c[u].y};
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_fp8x2_storage_t two = (__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1)));
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
      const int64_t e = (int64_t)row[u] * s.ld + (int64_t)blk[u] * kBlk + l16 * kLaneElems;
      if (s.vec && n[u] == 8) {
        if constexpr (DT == MB_F32) {
          float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + e);
          o[0] = make_float4(v[0], v[1], v[2], v[3]);
          o[1] = make_float4(v[4], v[5], v[6], v[7]);
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
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + e) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n[u]) store1<DT>(out, e + j, v[j]);
      }
    }
  }
}

// Rows and row lengths this file's index arithmetic covers: element offsets and
// block counts fit 62 bits.
bool shape_ok(int64_t rows, int64_t d, int64_t ld) {
  return rows >= 0 && d > 0 && ld >= d && ld <= ((int64_t)1 << 40) && rows <= ((int64_t)1 << 62) / ld;
}

Shape make_shape(int64_t rows, int64_t d, int64_t ld, const void* wide, int elem, const void* codes) {
  Shape s{rows, d, ld, (d + kBlk - 1) / kBlk, 0};
  s.vec = aligned(wide, 16) && (ld * elem) % 16 == 0 && aligned(codes, 8) && d % 8 == 0;
  return s;
}

template <typename K>
int act_grid(K fn, const Shape& s) {
  const int64_t per_cta = (int64_t)(kThreads / 16) * kUnroll;
  return grid_for(reinterpret_cast<const void*>(fn), (s.rows * s.blocks + per_cta - 1) / per_cta);
}

// 32-bit block indexes while the loop variable's overshoot (one grid stride past
// the end) cannot wrap: the division by blocks-per-row costs half as much.
bool small(const Shape& s) { return s.rows * s.blocks < ((int64_t)1 << 30); }

template <int DT>
int launch_pack(const void* x, const Shape& s, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  if (small(s)) {
    k_act_pack<DT, uint32_t><<<act_grid(&k_act_pack<DT, uint32_t>, s), kThreads, 0, st>>>(x, s, codes, scales);
  } else {
    k_act_pack<DT, int64_t><<<act_grid(&k_act_pack<DT, int64_t>, s), kThreads, 0, st>>>(x, s, codes, scales);
  }
  return cudaGetLastError() == cudaSuccess ? MB_OK : MB_ERR_CUDA;
}

template <int DT>
int launch_unpack(const uint8_t* codes, const uint8_t* scales, const Shape& s, void* out, cudaStream_t st) {
  if (small(s)) {
    k_act_unpack<DT, uint32_t><<<act_grid(&k_act_unpack<DT, uint32_t>, s), kThreads, 0, st>>>(codes, scales, s, out);
  } else {
    k_act_unpack<DT, int64_t><<<act_grid(&k_act_unpack<DT, int64_t>, s), kThreads, 0, st>>>(codes, scales, s, out);
  }
  return cudaGetLastError() == cudaSuccess ? MB_OK : MB_ERR_CUDA;
}

}  // namespace

int act_unpack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t d, void* out, int out_dtype,
               int64_t ld, cudaStream_t st) {
  if (!shape_ok(rows, d, ld)) return MB_ERR_ARG;
  if (rows == 0) return MB_OK;
  if (!codes || !scales || !out) return MB_ERR_ARG;
  switch (out_dtype) {
    case MB_F32: return launch_unpack<MB_F32>(codes, scales, make_shape(rows, d, ld, out, 4, codes), out, st);
    case MB_F16: return launch_unpack<MB_F16>(codes, scales, make_shape(rows, d, ld, out, 2, codes), out, st);
    case MB_BF16: return launch_unpack<MB_BF16>(codes, scales, make_shape(rows, d, ld, out, 2, codes), out, st);
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
  if (dtype == MB_F32) return launch_pack<MB_F32>(x, make_shape(rows, d, ld, x, 4, codes), codes, scales, st);
  if (dtype == MB_F16) return launch_pack<MB_F16>(x, make_shape(rows, d, ld, x, 2, codes), codes, scales, st);
  return launch_pack<MB_BF16>(x, make_shape(rows, d, ld, x, 2, codes), codes, scales, st);
}

MB_API int mb_act_unpack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t d, void* out,
                         int32_t out_dtype, int64_t ld, mb_stream_t stream) {
  return act_unpack(codes, scales, rows, d, out, out_dtype, ld, (cudaStream_t)stream);
}

}  // extern "C"
