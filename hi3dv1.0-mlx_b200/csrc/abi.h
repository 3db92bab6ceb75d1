// Host-side helpers shared by the entry points (not part of the public ABI).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hi3d_b200.h"

namespace hi3d {

// Record a formatted error message for hi3d_last_error_string(); returns `code`.
int set_error(int code, const char* fmt, ...);

// HI3D_OK, or HI3D_ERR_CUDA with the launch error recorded.
int check_launch(const char* what);

// Lets `kernel` use `bytes` of dynamic shared memory, once per kernel and device (`done`: the
// caller's flags for this kernel); HI3D_OK or HI3D_ERR_CUDA.
int allow_shared(const void* kernel, int bytes, bool (&done)[64], const char* what);

// Streaming multiprocessors of the current device (cached per device).
int sm_count();

// Encode a tiled TMA descriptor (dims/strides innermost first; strides are
// given for dims 1..rank-1 in bytes).
int encode_tmap(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims,
                const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swizzle);

// TMA descriptor of one attention operand, [batch][head][row][D] with the given element strides, boxes of
// 64 channels x box_rows rows (128-byte swizzle; attention.cu).
int make_attn_map(CUtensorMap* map, const void* base, int dtype, int D, int64_t rows, int heads, int64_t batch,
                  int64_t row_stride, int64_t head_stride, int64_t batch_stride, int box_rows);

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace hi3d
