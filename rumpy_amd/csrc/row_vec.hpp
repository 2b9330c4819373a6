// Rows of 8-element pieces in fp32, bf16 or fp16, at any element alignment: shared by residual_norm.hip and distill.hip.
#pragma once
#include "common.hpp"

template <int FMT> struct RowElem { typedef uint16_t type; };
template <> struct RowElem<RUMPY_FMT_F32> { typedef float type; };

// A row may start at any element (odd row lengths, slices of wider rows), so the 16-byte accesses are declared at element alignment: the
// hardware takes global dwordx4 accesses at any byte address and splits what crosses a cache line by itself.
typedef uint32_t row_u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) RowPiece16 { row_u32x4 v; };
struct __attribute__((packed, aligned(4))) RowPiece32 { row_u32x4 v; };

// 8 elements as they lie in memory: 16-bit formats fill `a` alone
template <int FMT> struct RowRaw { row_u32x4 a; };
template <> struct RowRaw<RUMPY_FMT_F32> { row_u32x4 a, b; };

template <int FMT> __device__ __forceinline__ float elem_to_f32(typename RowElem<FMT>::type v) {
  if constexpr (FMT == RUMPY_FMT_F32) return v;
  else if constexpr (FMT == RUMPY_FMT_F16) { union { uint16_t u; _Float16 h; } c; c.u = v; return (float)c.h; }
  else return bf16_bits_to_f32(v);
}
template <int FMT> __device__ __forceinline__ typename RowElem<FMT>::type f32_to_elem(float v) {
  if constexpr (FMT == RUMPY_FMT_F32) return v;
  else if constexpr (FMT == RUMPY_FMT_F16) { union { uint16_t u; _Float16 h; } c; c.h = (_Float16)v; return c.u; }
  else return f32_to_bf16_bits(v);
}
template <int FMT> __device__ __forceinline__ float load_elem(const void* base, size_t i) {
  return elem_to_f32<FMT>(reinterpret_cast<const typename RowElem<FMT>::type*>(base)[i]);
}

// the piece of 8 elements at p, of which n lie inside the row (n <= 0: nothing is read); elements outside hold `fill`'s bits
template <int FMT> __device__ __forceinline__ RowRaw<FMT> load_piece(const typename RowElem<FMT>::type* p, int n, float fill) {
  RowRaw<FMT> r;
  if constexpr (FMT == RUMPY_FMT_F32) {
    if (n >= 8) {
      r.a = reinterpret_cast<const RowPiece32*>(p)->v;
      r.b = reinterpret_cast<const RowPiece32*>(p + 4)->v;
    } else {
      const uint32_t f = __float_as_uint(fill);
#pragma unroll
      for (int i = 0; i < 4; ++i) { r.a[i] = i < n ? __float_as_uint(p[i]) : f; r.b[i] = 4 + i < n ? __float_as_uint(p[4 + i]) : f; }
    }
  } else {
    if (n >= 8) {
      r.a = reinterpret_cast<const RowPiece16*>(p)->v;
    } else {
      const uint32_t f = f32_to_elem<FMT>(fill);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = 2 * i < n ? p[2 * i] : f, hi = 2 * i + 1 < n ? p[2 * i + 1] : f;
        r.a[i] = lo | (hi << 16);
      }
    }
  }
  return r;
}
template <int FMT> __device__ __forceinline__ void unpack_piece(const RowRaw<FMT>& r, float (&o)[8]) {
  if constexpr (FMT == RUMPY_FMT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[i] = __uint_as_float(r.a[i]); o[4 + i] = __uint_as_float(r.b[i]); }
  } else if constexpr (FMT == RUMPY_FMT_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[2 * i] = elem_to_f32<FMT>((uint16_t)(r.a[i] & 0xffffu)); o[2 * i + 1] = elem_to_f32<FMT>((uint16_t)(r.a[i] >> 16)); }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[2 * i] = __uint_as_float(r.a[i] << 16); o[2 * i + 1] = __uint_as_float(r.a[i] & 0xffff0000u); }
  }
}
template <int FMT> __device__ __forceinline__ void load8(const void* base, size_t off, int n, float (&o)[8]) {
  unpack_piece<FMT>(load_piece<FMT>(reinterpret_cast<const typename RowElem<FMT>::type*>(base) + off, n, 0.f), o);
}
// rounds once, to nearest even
template <int FMT> __device__ __forceinline__ void store8(void* base, size_t off, int n, const float (&v)[8]) {
  typename RowElem<FMT>::type* p = reinterpret_cast<typename RowElem<FMT>::type*>(base) + off;
  if (n >= 8) {
    if constexpr (FMT == RUMPY_FMT_F32) {
      row_u32x4 a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = __float_as_uint(v[i]); b[i] = __float_as_uint(v[4 + i]); }
      reinterpret_cast<RowPiece32*>(p)->v = a;
      reinterpret_cast<RowPiece32*>(p + 4)->v = b;
    } else {
      row_u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = pack2<FMT>(v[2 * i], v[2 * i + 1]);
      reinterpret_cast<RowPiece16*>(p)->v = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < n) p[i] = f32_to_elem<FMT>(v[i]);
  }
}

// sum over LANES neighbouring lanes (a power of two up to 64), in every one of them: fixed order
template <int LANES> __device__ __forceinline__ float lanes_sum(float t, int lane) {
  if constexpr (LANES >= 2) t += dpp_quad1(t);
  if constexpr (LANES >= 4) t += dpp_quad2(t);
  if constexpr (LANES >= 8) t += dpp_half_mirror(t);
  if constexpr (LANES >= 16) t += dpp_row_mirror(t);
  if constexpr (LANES >= 32) t += lane_xor16(t, lane >> 4);
  if constexpr (LANES >= 64) t += lane_xor32(t, lane);
  return t;
}
