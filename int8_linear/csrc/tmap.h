// Host side of TMA: the driver's tensor-map encoder and 2-D tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "internal.h"

namespace i8l {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// Encodes a map.  The driver wants the thread to have a current context, which a thread that
// has launched nothing yet lacks: it gets that of its current device then.
template <typename... Args>
CUresult encode_tiled(EncodeTiledFn fn, Args... args) {
  CUresult r = fn(args...);
  int dev = 0;
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess)
    r = fn(args...);
  return r;
}

// Tensor map over a row-major 2-D matrix of `rows` x `cols` elements (row stride
// `ld_bytes`), boxes of box_cols x box_rows.
inline int make_map(CUtensorMap *map, CUtensorMapDataType type, const void *ptr, int64_t rows,
                    int64_t cols, int64_t ld_bytes, int box_cols, int box_rows,
                    CUtensorMapSwizzle swizzle, const char *what,
                    CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_NONE) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(I8L_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld_bytes)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_tiled(fn, map, type, 2u, const_cast<void *>(ptr), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(I8L_ECUDA, "cuTensorMapEncodeTiled failed (CUresult %d) for the %s map [%lld x %lld]",
                     static_cast<int>(r), what, static_cast<long long>(rows),
                     static_cast<long long>(cols));
  return I8L_OK;
}

}  // namespace i8l
