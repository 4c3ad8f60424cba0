// Appending keys and values to the 4-bit paged cache, queries and keys rotated on the way, and reading rows back.
//
// A step's queries, keys and values are read once and written once: 2 bytes an element in, 2 out for the queries and
// half a byte (+ 4 bytes a head) for keys and values.  There is no reuse, so memory bounds a prompt and the launch a
// decode step; as separate elementwise steps the same work takes some thirty launches.
#include "kv4_cache.h"

namespace {

using namespace serving;

constexpr int kThreads = 256;

struct AppendArgs {
  const void *query, *key, *value;
  long long q_token, q_head, k_token, k_head, v_token, v_head;
  const float* cos_sin;
  long long cs_stride;
  const int64_t *pos, *slots;
  void* out;
  uint8_t* cache;
  int tokens, heads, kv_heads, rotary, interleaved, block_size, token_shift;
  long long positions, slots_in_cache;
};

template <typename T>
struct Vec8;
template <>
struct Vec8<f16> {
  typedef f16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Vec8<bf16> {
  typedef bf16 type __attribute__((ext_vector_type(8)));
};

// Least and largest of the 2 x 8 values that each of the L lanes of a row holds.
template <int L>
__device__ __forceinline__ void row_range(float& least, float& most) {
#pragma unroll
  for (int m = 1; m < L; m <<= 1) {
    least = fminf(least, __shfl_xor(least, m));
    most = fmaxf(most, __shfl_xor(most, m));
  }
}

// 8 codes of a word.  The same operations in the same order as the format defines them (no product is fused into a
// sum), so that every caller finds the codes that the definition gives.
__device__ __forceinline__ uint32_t encode(const float* x, float least, float scale) {
#pragma clang fp contract(off)
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(__builtin_rintf((x[i] - least) / scale), 0.f), 15.f);
    w |= (uint32_t)c << (4 * i);
  }
  return w;
}

// L = D / 16 lanes work on one head of one token, each on two pieces of 8 elements: the two halves of its rotated
// pairs (or two neighbouring pieces), so that a rotation needs no other lane.  A workgroup belongs to one token (to
// several whose heads do not fill it) and walks over its heads, so that a lane reads its angles once.  What is read here
// is read once and what the queries become is written once: both pass the caches by, which leaves these to the lines of
// the cache that neighbouring tokens share.
// 8192 tokens of 64 + 8 heads of 128, bf16: 59 us, 5.3 TB/s (66 with 16 tokens a workgroup, 70 with these through the
// caches).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(AppendArgs a) {
#pragma clang fp contract(off)
  typedef typename Vec8<T>::type vec8;
  constexpr int L = D / 16;
  constexpr int kRows = kThreads / L;
  const int lane = threadIdx.x % L, row = threadIdx.x / L;
  const int t = (blockIdx.x << a.token_shift) + (row & ((1 << a.token_shift) - 1));
  const int head_step = (kRows >> a.token_shift) * gridDim.y;
  int head = blockIdx.y * (kRows >> a.token_shift) + (row >> a.token_shift);
  const int all = a.heads + 2 * a.kv_heads;
  if (t >= a.tokens || head >= all) return;  // (whole rows leave; the lanes of a row stay together)

  const long long slot = a.slots[t];
  const bool stores = slot >= 0 && slot < a.slots_in_cache;
  const int nr = a.rotary / 16;
  const bool turns = lane < nr;
  const int first = turns && !a.interleaved ? lane : 2 * lane;
  const int second = turns && !a.interleaved ? lane + nr : 2 * lane + 1;
  float co[8], si[8];
  if (turns) {
    const long long p = a.pos[t];
    if (p >= 0 && p < a.positions) {
      const float* angles = a.cos_sin + p * a.cs_stride + 8 * lane;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const f32x4 c = *reinterpret_cast<const f32x4*>(angles + i);
        const f32x4 s = *reinterpret_cast<const f32x4*>(angles + a.rotary / 2 + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) co[i + j] = c[j], si[i + j] = s[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) co[i] = si[i] = __builtin_nanf("");
    }
  }
  const long long block = stores ? slot / a.block_size : 0;
  const int place = stores ? (int)(slot - block * a.block_size) : 0;

  for (; head < all; head += head_step) {
    const bool is_q = head < a.heads, is_v = head >= a.heads + a.kv_heads;
    if (!is_q && !stores) break;
    const T* src;
    if (is_q)
      src = static_cast<const T*>(a.query) + t * a.q_token + head * a.q_head;
    else if (!is_v)
      src = static_cast<const T*>(a.key) + t * a.k_token + (head - a.heads) * a.k_head;
    else
      src = static_cast<const T*>(a.value) + t * a.v_token + (head - a.heads - a.kv_heads) * a.v_head;
    const int pa = is_v ? lane : first, pb = is_v ? lane + L : second;
    const vec8 va = __builtin_nontemporal_load(reinterpret_cast<const vec8*>(src + 8 * pa));
    const vec8 vb = __builtin_nontemporal_load(reinterpret_cast<const vec8*>(src + 8 * pb));
    float x[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)va[i], x[8 + i] = (float)vb[i];
    if (turns && !is_v) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = x[2 * i], q = x[2 * i + 1];
          x[2 * i] = p * co[i] - q * si[i];
          x[2 * i + 1] = q * co[i] + p * si[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = x[i], q = x[8 + i];
          x[i] = p * co[i] - q * si[i];
          x[8 + i] = q * co[i] + p * si[i];
        }
      }
    }
    if (is_q) {
      T* dst = static_cast<T*>(a.out) + ((long long)t * a.heads + head) * D;
      vec8 ra, rb;
#pragma unroll
      for (int i = 0; i < 8; ++i) ra[i] = (T)x[i], rb[i] = (T)x[8 + i];
      __builtin_nontemporal_store(ra, reinterpret_cast<vec8*>(dst + 8 * pa));
      __builtin_nontemporal_store(rb, reinterpret_cast<vec8*>(dst + 8 * pb));
      continue;
    }
    float lo = x[0], hi = x[0];
    bool nan = x[0] != x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]), nan |= x[i] != x[i];
    if (nan) hi = __builtin_inff();  // (min and max pass a NaN by)
    row_range<L>(lo, hi);
    f16 least = (f16)lo;
    float step = (hi - (float)least) * (1.f / 15.f);
    asm("" : "+v"(step));  // (rounded to fp32 before it is to fp16: one instruction would do both at once)
    f16 scale = (f16)step;
    const bool held = __builtin_isfinite((float)least) && __builtin_isfinite((float)scale);
    uint32_t wa = 0, wb = 0;
    if (held && (float)scale > 0.f) {
      wa = encode(x, (float)least, (float)scale);
      wb = encode(x + 8, (float)least, (float)scale);
    }
    if (!held) least = scale = (f16)__builtin_nanf("");
    const int kv = head - a.heads - (is_v ? a.kv_heads : 0);
    uint8_t* base = a.cache + (block * a.kv_heads + kv) * Kv4<D>::block_bytes(a.block_size);
    uint8_t* codes;
    int piece;  // bytes from one piece of a token to the next
    if (is_v) {
      codes = base + Kv4<D>::values(a.block_size) + (place / 16) * Kv4<D>::kGroupBytes + (place % 16) * 4;
      piece = Kv4<D>::kPieceBytes;
    } else {
      codes = base + place * Kv4<D>::kTokenBytes;
      piece = 4;
    }
    *reinterpret_cast<uint32_t*>(codes + pa * piece) = wa;
    *reinterpret_cast<uint32_t*>(codes + pb * piece) = wb;
    if (lane == 0) {
      const int at = (is_v ? Kv4<D>::value_params(a.block_size) : Kv4<D>::key_params(a.block_size)) + 4 * place;
      *reinterpret_cast<f16x2*>(base + at) = f16x2{scale, least};
    }
  }
}

// One lane a piece of 8 elements: a word of codes and the token's parameters in, 16 bytes out.  42 MB of 8192 tokens of 8
// heads of 128 in 12.5 us, 3.4 TB/s: loads of 4 bytes, and each token's parameters once for every piece, bound it.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const uint8_t* __restrict__ cache, const int64_t* __restrict__ slots,
                                                        T* __restrict__ key, T* __restrict__ value, long long pieces,
                                                        int kv_heads, int block_size, long long slots_in_cache) {
  typedef typename Vec8<T>::type vec8;
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= pieces) return;
  const int piece = (int)(i % (D / 8));
  const long long head_row = i / (D / 8);
  const long long row = head_row / kv_heads;
  const int head = (int)(head_row - row * kv_heads);
  const long long slot = slots[row];
  vec8 k = {}, v = {};
  if (slot >= 0 && slot < slots_in_cache) {
    const long long block = slot / block_size;
    const int place = (int)(slot - block * block_size);
    const uint8_t* base = cache + (block * kv_heads + head) * Kv4<D>::block_bytes(block_size);
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(base + place * Kv4<D>::kTokenBytes + 4 * piece);
    const uint32_t vw = *reinterpret_cast<const uint32_t*>(base + Kv4<D>::values(block_size) + (place / 16) * Kv4<D>::kGroupBytes +
                                                           piece * Kv4<D>::kPieceBytes + (place % 16) * 4);
    const f16x2 kp = *reinterpret_cast<const f16x2*>(base + Kv4<D>::key_params(block_size) + 4 * place);
    const f16x2 vp = *reinterpret_cast<const f16x2*>(base + Kv4<D>::value_params(block_size) + 4 * place);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      k[e] = (T)__builtin_fmaf((float)((kw >> (4 * e)) & 15u), (float)kp.x, (float)kp.y);
      v[e] = (T)__builtin_fmaf((float)((vw >> (4 * e)) & 15u), (float)vp.x, (float)vp.y);
    }
  }
  *reinterpret_cast<vec8*>(key + i * 8) = k;
  *reinterpret_cast<vec8*>(value + i * 8) = v;
}

thread_local int g_last_hip_error = 0;

}  // namespace

extern "C" SERVING_HIDDEN int serving_after_launch() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return SERVING_OK;
  g_last_hip_error = (int)e;
  return SERVING_E_LAUNCH;
}

extern "C" int serving_last_hip_error(void) { return g_last_hip_error; }

extern "C" int serving_abi_version(void) { return SERVING_ABI_VERSION; }

extern "C" const char* serving_strerror(int code) {
  switch (code) {
    case SERVING_OK: return "ok";
    case SERVING_E_NULL: return "null pointer argument";
    case SERVING_E_SHAPE: return "a size is out of its range, or sizes do not fit each other";
    case SERVING_E_HEAD: return "head_size must be 64 or 128";
    case SERVING_E_BLOCK: return "block_size must be a multiple of 16 from 16 to 4096";
    case SERVING_E_ROTARY: return "the rotated part of a head must be a multiple of 16 elements and no larger than a head";
    case SERVING_E_ALIGN: return "pointers must be 16-byte aligned and strides multiples of 8 elements";
    case SERVING_E_LAUNCH: return "HIP launch failed";
    case SERVING_E_TOO_LARGE: return "too large for one launch";
    case SERVING_E_WORKSPACE: return "workspace too small";
    default: return "unknown serving error";
  }
}

extern "C" size_t serving_kv4_cache_bytes(long long num_blocks, int block_size, int kv_heads, int head_size) {
  if (num_blocks <= 0 || num_blocks > 0x7fffffffLL || kv_heads <= 0 || kv_heads > 65535 || !head_size_ok(head_size) ||
      !block_size_ok(block_size))
    return 0;
  return (size_t)num_blocks * kv_heads * block_size * (head_size + 8);
}

extern "C" int serving_rope_append_kv4(const void* query, long long q_token, long long q_head, const void* key,
                                       long long k_token, long long k_head, const void* value, long long v_token,
                                       long long v_head, const float* cos_sin, long long cs_stride, const int64_t* pos,
                                       const int64_t* slots, void* out, void* cache, int tokens, int heads, int kv_heads,
                                       int head_size, int rotary, int interleaved, long long positions,
                                       long long num_blocks, int block_size, int bf16_in, void* stream) {
  if (!query || !key || !value || !slots || !out || !cache || (rotary > 0 && (!cos_sin || !pos))) return SERVING_E_NULL;
  if (!head_size_ok(head_size)) return SERVING_E_HEAD;
  if (!block_size_ok(block_size)) return SERVING_E_BLOCK;
  if (rotary < 0 || rotary % 16 || rotary > head_size) return SERVING_E_ROTARY;
  if (tokens <= 0 || heads <= 0 || heads > 65535 || kv_heads <= 0 || kv_heads > 65535 || positions < 0 ||
      num_blocks <= 0 || num_blocks > 0x7fffffffLL)
    return SERVING_E_SHAPE;
  if (tokens > (1 << 30)) return SERVING_E_TOO_LARGE;
  if (!aligned16(query) || !aligned16(key) || !aligned16(value) || !aligned16(out) || !aligned16(cache) ||
      !aligned16(cos_sin) || (q_token | q_head | k_token | k_head | v_token | v_head) % 8 || cs_stride % 4)
    return SERVING_E_ALIGN;
  AppendArgs a{query,      key,     value,      q_token,      q_head,     k_token,    k_head, v_token,
               v_head,     cos_sin, cs_stride,  pos,          slots,      out,        static_cast<uint8_t*>(cache),
               tokens,     heads,   kv_heads,   rotary,       interleaved, block_size, 0,     positions,
               num_blocks * block_size};
  const int all = heads + 2 * kv_heads;
  int per_pass = kThreads / (head_size / 16);  // heads of a token that a workgroup takes at once
  while (per_pass >= 2 * all) per_pass /= 2, ++a.token_shift;
  const int x = (tokens + (1 << a.token_shift) - 1) >> a.token_shift;
  if (x > 0xffffff) return SERVING_E_TOO_LARGE;  // (a grid has less than 2^32 threads in a direction)
  const int passes = (all + per_pass - 1) / per_pass;
  // as many workgroups as fill the chip a few times over, and no more: each reads its token's angles once
  int y = (2048 + x - 1) / x;
  y = y > passes ? passes : y;
  y = y > 65535 ? 65535 : y;
  const dim3 grid((unsigned)x, (unsigned)y);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_size == 64) {
    if (bf16_in)
      hipLaunchKernelGGL((rope_append_kernel<bf16, 64>), grid, dim3(kThreads), 0, s, a);
    else
      hipLaunchKernelGGL((rope_append_kernel<f16, 64>), grid, dim3(kThreads), 0, s, a);
  } else {
    if (bf16_in)
      hipLaunchKernelGGL((rope_append_kernel<bf16, 128>), grid, dim3(kThreads), 0, s, a);
    else
      hipLaunchKernelGGL((rope_append_kernel<f16, 128>), grid, dim3(kThreads), 0, s, a);
  }
  return serving_after_launch();
}

extern "C" int serving_read_kv4(const void* cache, const int64_t* slots, void* key, void* value, long long rows,
                                int kv_heads, int head_size, long long num_blocks, int block_size, int bf16_out,
                                void* stream) {
  if (!cache || !slots || !key || !value) return SERVING_E_NULL;
  if (!head_size_ok(head_size)) return SERVING_E_HEAD;
  if (!block_size_ok(block_size)) return SERVING_E_BLOCK;
  if (rows <= 0 || kv_heads <= 0 || kv_heads > 65535 || num_blocks <= 0 || num_blocks > 0x7fffffffLL) return SERVING_E_SHAPE;
  if (!aligned16(cache) || !aligned16(key) || !aligned16(value)) return SERVING_E_ALIGN;
  if (rows > (1LL << 40)) return SERVING_E_TOO_LARGE;
  const long long pieces = rows * kv_heads * (head_size / 8);
  const long long groups = (pieces + kThreads - 1) / kThreads;
  if (groups > 0xffffff) return SERVING_E_TOO_LARGE;
  const dim3 grid((unsigned)groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint8_t* c = static_cast<const uint8_t*>(cache);
  const long long have = num_blocks * block_size;
#define SERVING_READ(T, D)                                                                                            \
  hipLaunchKernelGGL((read_kernel<T, D>), grid, dim3(kThreads), 0, s, c, slots, static_cast<T*>(key),                 \
                     static_cast<T*>(value), pieces, kv_heads, block_size, have)
  if (head_size == 64) {
    if (bf16_out)
      SERVING_READ(bf16, 64);
    else
      SERVING_READ(f16, 64);
  } else {
    if (bf16_out)
      SERVING_READ(bf16, 128);
    else
      SERVING_READ(f16, 128);
  }
#undef SERVING_READ
  return serving_after_launch();
}
