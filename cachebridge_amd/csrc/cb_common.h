// What every source of the library shares: the error text of the last failed
// call, address-space pointers, bf16 packing and the device form of cb_rows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "../../include/cachebridge_hip.h"

// The message cb_last_error returns: one per thread for the whole library.
inline thread_local std::string g_last_error;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

#define CB_HIP(expr)                                                                       \
  do {                                                                                     \
    hipError_t e_ = (expr);                                                                \
    if (e_ != hipSuccess) return fail(CB_EHIP, "%s: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Global-address-space pointers. Generic (flat) loads and stores also count
// against the LDS wait counter, which would make every LDS wait drain all
// outstanding HBM traffic, so every pool/table access goes through these.
#if defined(__HIP_DEVICE_COMPILE__)
#define CB_GLOBAL __attribute__((address_space(1)))
#define CB_CONST __attribute__((address_space(4)))
#define CB_LDS __attribute__((address_space(3)))
#else
#define CB_GLOBAL
#define CB_CONST
#define CB_LDS
#endif
typedef const CB_GLOBAL char* gcptr;
typedef CB_GLOBAL char* gptr;
template <typename V>
__device__ inline V gload(gcptr p) {
  return *reinterpret_cast<const CB_GLOBAL V*>(p);
}
template <typename V>
__device__ inline void gstore(gptr p, const V& v) {
  *reinterpret_cast<CB_GLOBAL V*>(p) = v;
}
// Plan metadata (job, unit and pair tables, layer pointer arrays) is read-only
// for a launch: loading it through the constant address space lets the
// compiler use scalar loads for wave-uniform indices instead of vector loads
// whose results would have to wait for every older vector load.
template <typename V>
__device__ inline V cload(const V* p) {
  return *(const CB_CONST V*)(p);
}
__device__ inline gcptr as_global(const void* p) { return (gcptr)p; }
__device__ inline gptr as_global(void* p) { return (gptr)p; }
__device__ inline const CB_GLOBAL float* gtab(const float* p) { return (const CB_GLOBAL float*)p; }

constexpr int kWave = 64;

__device__ inline float lo_bf(uint32_t w) { return __uint_as_float(w << 16); }
__device__ inline float hi_bf(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Two fp32 -> packed bf16 pair, round to nearest even (v_cvt_pk_bf16_f32).
__device__ inline uint32_t pack_bf16(float a, float b) {
  const f32x2 f = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

struct DevRows {
  const void* const* k_layers;
  const void* const* v_layers;
  const char* k_base;
  const char* v_base;
  int64_t layer_stride_b;
  int64_t row_stride_b;
  int64_t rows;
  const void* index;
  int64_t index_offset;
  int32_t index_kind;
  int32_t page_size;
  int32_t head_offset;
  int32_t layers;
};

__device__ inline gcptr layer_base(const DevRows& R, int kind, int layer) {
  const void* const* arr = kind ? R.v_layers : R.k_layers;
  if (arr) return as_global(cload(arr + layer));
  return as_global(kind ? R.v_base : R.k_base) + layer * R.layer_stride_b;
}

// align: the byte alignment the launch needs of strides and bases (16 for the
// vector kernels, one element for the generic kernel).
int to_dev_rows(const cb_rows& r, int elem_bytes, DevRows* out, int align = 16) {
  out->k_layers = r.k_layers;
  out->v_layers = r.v_layers;
  out->k_base = static_cast<const char*>(r.k_base);
  out->v_base = static_cast<const char*>(r.v_base);
  out->layer_stride_b = r.layer_stride * elem_bytes;
  out->row_stride_b = r.row_stride * elem_bytes;
  out->rows = r.rows;
  out->index = r.index;
  out->index_offset = r.index_offset;
  out->index_kind = r.index_kind;
  out->page_size = r.page_size;
  out->head_offset = r.head_offset;
  out->layers = r.num_layers;
  if (r.index_kind < CB_INDEX_IDENTITY || r.index_kind > CB_INDEX_BLOCK_TABLE)
    return fail(CB_EINVAL, "unknown index_kind %d", r.index_kind);
  if (r.index_kind != CB_INDEX_IDENTITY && !r.index)
    return fail(CB_EINVAL, "index pointer required for index_kind %d", r.index_kind);
  if (r.index_kind == CB_INDEX_BLOCK_TABLE && r.page_size <= 0)
    return fail(CB_EINVAL, "block table needs page_size > 0");
  if (r.index_offset < 0 || r.index_offset > (int64_t{1} << 30))
    return fail(CB_EINVAL, "index_offset out of range");
  if (r.rows <= 0) return fail(CB_EINVAL, "rows must be > 0");
  if (!r.k_layers && (!r.k_base || !r.v_base))
    return fail(CB_EINVAL, "either per-layer pointer arrays or k_base/v_base are required");
  if (r.k_layers && !r.v_layers) return fail(CB_EINVAL, "v_layers required with k_layers");
  if ((out->row_stride_b % align) || (out->layer_stride_b % align))
    return fail(CB_EINVAL, "row and layer strides must be multiples of %d bytes", align);
  if ((reinterpret_cast<uintptr_t>(r.k_base) | reinterpret_cast<uintptr_t>(r.v_base)) % align)
    return fail(CB_EINVAL, "k_base/v_base must be %d-byte aligned", align);
  return CB_OK;
}

}  // namespace
