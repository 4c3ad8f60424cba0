// The paged cache of keys and values in 4 bits: where a block keeps what, and the types the kernels on it share.
// (The format is defined in include/serving_ops.h.)
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/serving_ops.h"

#define SERVING_HIDDEN __attribute__((visibility("hidden")))

// Records the hipError_t of a failed launch for serving_last_hip_error() (kv4_append.hip).
extern "C" SERVING_HIDDEN int serving_after_launch();

namespace SERVING_HIDDEN serving {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// What a block holds of one head, in bytes.
template <int D>
struct Kv4 {
  static constexpr int kTokenBytes = D / 2;     // of a token's keys, or values
  static constexpr int kPieceBytes = 64;        // one piece (8 elements) of the values of 16 tokens
  static constexpr int kGroupBytes = 8 * D;     // the values of 16 tokens
  static constexpr long long block_bytes(int p) { return (long long)p * (D + 8); }
  static constexpr int values(int p) { return p * kTokenBytes; }
  static constexpr int key_params(int p) { return p * D; }
  static constexpr int value_params(int p) { return p * D + 4 * p; }
};

inline bool head_size_ok(int d) { return d == 64 || d == 128; }
inline bool block_size_ok(int p) { return p > 0 && p % 16 == 0 && p <= 4096; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace serving
