// Log probabilities of given tokens, the entropy of each row and its most likely tokens, in one pass over the logits.
//
// A row (or, of a long one, a segment) is read once into the registers of one workgroup, which then takes from there
// its maximum m, the sums  Z - 1 = sum exp(x - m) - 1  and  sum exp(x - m) (x - m),  and its largest elements.  Memory
// bounds it: 2 or 4 bytes an element against about a dozen vector instructions.
//   log p_t = x_t - m - log Z,   H = log Z - sum exp(x - m) (x - m) / Z    (both terms of H are positive: no cancellation)
// Z - 1 is summed without the maxima themselves, so that log1p keeps its digits where one token has nearly all the
// probability.
// The n largest: the maxima of 64 disjoint groups of elements are ranked by one wave; the n-th of them bounds the n-th
// largest element from below, so only elements not below it (little more than n) go to LDS, where each counts those
// ahead of it.  Equal elements are told apart by their index, which makes the order total and the result one of its own.
#include "kv4_cache.h"

#include <type_traits>

namespace {

using namespace serving;

constexpr int kMaxTop = 64;       // groups that are ranked for the bound
constexpr int kCandidates = 1024;  // elements not below the bound that LDS takes; more (rows of equals) go the long way

constexpr int kFewRows = 256;  // a workgroup of 1024 lanes for each CU, or four of 512
constexpr int kMaxVocab = 64 * 32760;  // 64 segments: a lane of the join each, and their keys in LDS

typedef unsigned long long u64;

// What a segment leaves of itself for the join: its maximum, how often it occurs, the sums without it.
struct Part {
  float most, rest, weighted;
  int count;
};

template <int TYPE>  // 0 fp16, 1 bf16, 2 fp32
struct Logits {
  static constexpr int kEach = TYPE == 2 ? 4 : 8;  // elements of 16 bytes
  static constexpr int kBytes = TYPE == 2 ? 4 : 2;
  static __device__ __forceinline__ float get(const u32x4& v, int i) {
    const uint32_t w = v[TYPE == 2 ? i : i / 2];  // (a bit cast of a vector's element itself takes the first one)
    if (TYPE == 2) return __builtin_bit_cast(float, w);
    if (TYPE == 1) return __builtin_bit_cast(float, i & 1 ? w & 0xffff0000u : w << 16);
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    return (float)(i & 1 ? h.y : h.x);
  }
  static __device__ __forceinline__ void hide(u32x4& v, int i) {  // element i becomes -inf
    if (TYPE == 2) {
      v[i] = 0xff800000u;
    } else {
      const uint32_t inf = TYPE == 1 ? 0xff80u : 0xfc00u;
      v[i / 2] = i & 1 ? (v[i / 2] & 0xffffu) | (inf << 16) : (v[i / 2] & 0xffff0000u) | inf;
    }
  }
};

// A number that orders as the value does: both zeros alike, a NaN above +inf.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x != x ? __builtin_nanf("") : x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ u64 key_of(float x, int index) {
  return ((u64)ordered(x) << 32) | (uint32_t)(0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ int index_of(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }

__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // NaN if one is

template <typename V, typename F>
__device__ __forceinline__ V wave_all(V v, F f) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = f(v, __shfl_xor(v, m));
  return v;
}

// log Z and H from the maximum's count, the rest of Z and the weighted sum.
__device__ __forceinline__ void finish(double count, double rest, double weighted, double& log_z, double& entropy) {
  log_z = count == 1.0 ? log1p(rest) : log(count + rest);
  entropy = log_z - weighted / (count + rest);
}

struct Args {
  const uint8_t* logits;
  long long row_stride;  // bytes
  const int64_t* token_ids;
  float *logprob, *entropy;
  int64_t* top_ids;
  float* top_logprobs;
  Part* parts;  // [rows][segments], and behind them the keys [rows][segments][top]
  u64* keys;
  int vocab, top, segments, segment;
};

template <int TYPE, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS, 4) logprobs_kernel(Args a) {
  typedef Logits<TYPE> X;
  constexpr int kWaves = THREADS / 64;
  constexpr float kLog2e = 1.44269504088896340736f;
  __shared__ uint32_t lane_most[kWaves][64];
  __shared__ float sums[kWaves][2];
  __shared__ int counts[kWaves];
  __shared__ u64 candidates[kCandidates];
  __shared__ u64 wave_best[kWaves];
  __shared__ int n_candidates;
  __shared__ int groups_ahead[64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / a.segments, seg = blockIdx.x - row * a.segments;
  const int begin = seg * a.segment;                         // of this segment in its row
  const int size = min(a.segment, a.vocab - begin);
  const uint8_t* row_base = a.logits + row * a.row_stride;
  const uint8_t* base = row_base + (long long)begin * X::kBytes;
  const int skip = (int)((reinterpret_cast<uintptr_t>(base) & 15u) / X::kBytes);  // of the first 16 bytes, not ours
  const u32x4* words = reinterpret_cast<const u32x4*>(base - skip * X::kBytes);
  if (tid == 0) n_candidates = 0;
  if (tid < 64) groups_ahead[tid] = 0;

  const auto fetch = [&](int k) {
    const int e = (k * THREADS + tid) * X::kEach - skip;  // of this lane's first element in the segment
    u32x4 w = {0u, 0u, 0u, 0u};
    // (16 aligned bytes that hold one of the row's elements: never outside the pages of its tensor)
    const bool some = e < size && e > -X::kEach;
    if (some) w = words[k * THREADS + tid];
    if (!some || e < 0 || e + X::kEach > size) {
#pragma unroll
      for (int i = 0; i < X::kEach; ++i)
        if (e + i < 0 || e + i >= size) X::hide(w, i);
    }
    return w;
  };
  u32x4 v[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = fetch(k);
  float given = 0.f;
  long long token = -1;
  if (a.segments == 1 && tid == 0) {
    token = a.token_ids[row];
    if (token >= 0 && token < a.vocab) {
      const uint8_t* p = row_base + token * X::kBytes;
      given = TYPE == 2 ? *reinterpret_cast<const float*>(p)
                        : TYPE == 1 ? __builtin_bit_cast(float, (uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16)
                                    : (float)*reinterpret_cast<const f16*>(p);
    }
  }

  float mine = -__builtin_inff();
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < X::kEach; ++i) mine = larger(mine, X::get(v[k], i));
  lane_most[wave][lane] = ordered(mine);
  __syncthreads();
  // the 64 groups: the elements of equal lanes of all waves
  uint32_t group = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) group = max(group, lane_most[w][lane]);
  const float most = unordered(wave_all(group, [](uint32_t p, uint32_t q) { return max(p, q); }));

  float rest = 0.f, weighted = 0.f;
  int count = 0;
  const auto sum = [&](auto with_maximum) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < X::kEach; ++i) {
        const float d = fmaxf(X::get(v[k], i) - most, -10000.f) * kLog2e;  // (-inf adds nothing, and not 0 * inf)
        const float p = __builtin_amdgcn_exp2f(d);
        if (with_maximum) {
          count += d == 0.f;
          rest += d == 0.f ? 0.f : p;
        } else {
          rest += p;
        }
        weighted = __builtin_fmaf(p, d, weighted);
      }
      __builtin_amdgcn_sched_barrier(0);  // (16 bytes at a time: more at once would only take registers)
    }
  };
  if (__any(mine == most)) {  // the wave or two that hold a maximum
    asm volatile("");  // (keeps this a branch)
    sum(std::true_type());
  } else {
    sum(std::false_type());
  }
  weighted *= 0.69314718055994530942f;
  rest = wave_all(rest, [](float p, float q) { return p + q; });
  weighted = wave_all(weighted, [](float p, float q) { return p + q; });
  count = wave_all(count, [](int p, int q) { return p + q; });
  if (lane == 0) sums[wave][0] = rest, sums[wave][1] = weighted, counts[wave] = count;

  // The n-th largest group maximum: each lane counts the groups ahead of its own, a share of them in each wave (told
  // apart by the lane in the last six bits; what these held only lowers the bound).
  const uint32_t own = (group & ~63u) | (uint32_t)(63 - lane);
  if (a.top > 0) {
    int ahead = 0;
#pragma unroll
    for (int i = 0; i < 64 / kWaves; ++i)
      ahead += (uint32_t)__builtin_amdgcn_readlane(own, __builtin_amdgcn_readfirstlane(wave) * (64 / kWaves) + i) > own;
    atomicAdd(&groups_ahead[lane], ahead);
  }
  __syncthreads();
  if (a.top > 0) {
    const uint32_t bound = __builtin_amdgcn_readlane(own, __builtin_ctzll(__ballot(groups_ahead[lane] == a.top - 1))) & ~63u;
    const float border = bound < ordered(-__builtin_inff()) ? -__builtin_inff() : unordered(bound);
    if (most != most) {  // a row with a NaN: ordered numbers know where it stands, comparisons do not
#pragma unroll 1
      for (int k = 0; k < NV; ++k) {
        const u32x4 w = fetch(k);
        for (int i = 0; i < X::kEach; ++i) {
          const float x = X::get(w, i);
          const int e = (k * THREADS + tid) * X::kEach - skip + i;
          if (ordered(x) >= bound && e >= 0 && e < size) {
            const int at = atomicAdd(&n_candidates, 1);
            if (at < kCandidates) candidates[at] = key_of(x, begin + e);
          }
        }
      }
    } else if (mine >= border) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        bool some = false;
#pragma unroll
        for (int i = 0; i < X::kEach; ++i) some |= X::get(v[k], i) >= border;
        if (!some) continue;
        const int e = (k * THREADS + tid) * X::kEach - skip;
#pragma unroll
        for (int i = 0; i < X::kEach; ++i) {
          const float x = X::get(v[k], i);
          if (x >= border && e + i >= 0 && e + i < size) {
            const int at = atomicAdd(&n_candidates, 1);
            if (at < kCandidates) candidates[at] = key_of(x, begin + e + i);
          }
        }
      }
    }
  }
  __syncthreads();

  float all_rest = 0.f, all_weighted = 0.f;
  int all_count = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all_rest += sums[w][0], all_weighted += sums[w][1], all_count += counts[w];
  const bool finite = __builtin_isfinite(most);
  const int n = n_candidates;
  double log_z = 0.0, entropy = 0.0;
  const long long part = (long long)row * a.segments + seg;
  if (a.segments == 1) {
    if (finite) finish(all_count, all_rest, all_weighted, log_z, entropy);
    if (!finite) log_z = entropy = __builtin_nan("");
    if (tid == 0) {
      a.logprob[row] = token >= 0 && token < a.vocab ? (float)((double)(given - most) - log_z) : __builtin_nanf("");
      a.entropy[row] = (float)entropy;
    }
  } else if (tid == 0) {
    a.parts[part] = Part{most, all_rest, all_weighted, all_count};
  }
  const auto place = [&](int rank, u64 key) {
    if (a.segments == 1) {
      a.top_ids[(long long)row * a.top + rank] = index_of(key);
      a.top_logprobs[(long long)row * a.top + rank] =
          (float)((double)(unordered((uint32_t)(key >> 32)) - most) - log_z);
    } else {
      a.keys[part * a.top + rank] = key;
    }
  };
  const int want = min(a.top, size);
  if (a.segments > 1)
    for (int r = want + tid; r < a.top; r += THREADS) a.keys[part * a.top + r] = 0;  // (below every element's key)
  if (n <= kCandidates) {
    for (int i = tid; i < n; i += THREADS) {
      const u64 key = candidates[i];
      int ahead = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) ahead += candidates[j] > key;
      if (ahead < want) place(ahead, key);
    }
    return;
  }
  // Too many equals at the bound: one rank after the other over all elements.
  u64 last = ~0ull;
  for (int r = 0; r < want; ++r) {
    u64 best = 0;
#pragma unroll 1
    for (int k = 0; k < NV; ++k) {
      const u32x4 w = fetch(k);
      const int e = (k * THREADS + tid) * X::kEach - skip;
#pragma unroll
      for (int i = 0; i < X::kEach; ++i) {
        const u64 key = key_of(X::get(w, i), begin + e + i);
        if (e + i >= 0 && e + i < size && key < last && key > best) best = key;
      }
    }
    best = wave_all(best, [](u64 p, u64 q) { return p > q ? p : q; });
    if (lane == 0) wave_best[wave] = best;
    __syncthreads();
    last = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) last = last > wave_best[w] ? last : wave_best[w];
    if (tid == 0) place(r, last);
    __syncthreads();
  }
}

// Joins the segments of a row: sums by one wave, a lane a segment, the most likely tokens by counting the keys ahead
// of each.  Four rows a workgroup, a wave each, where there are many rows with few keys (4096 rows of 80 keys 10 us
// against 18; 64 of them 7 against 4.5).
template <int TYPE, int ROWS>
__global__ void __launch_bounds__(256) join_kernel(Args a, int rows) {
  typedef Logits<TYPE> X;
  constexpr int kLanes = 256 / ROWS, kKeys = ROWS == 1 ? 4096 : 128, kRanked = ROWS == 1 ? 512 : 128;
  __shared__ double shared_log_z[ROWS];
  __shared__ float shared_most[ROWS];
  __shared__ u64 all_keys[ROWS][kKeys], ranked[ROWS][kRanked], bound[ROWS];
  __shared__ int n_ranked[ROWS];
  const int which = threadIdx.x / kLanes, tid = threadIdx.x % kLanes;
  const int row = blockIdx.x * ROWS + which;
  const bool on = row < rows;
  const Part* parts = a.parts + (long long)row * a.segments;
  const int n = on ? a.segments * a.top : 0;
  u64* keys = all_keys[which];
  if (tid == 0) n_ranked[which] = 0, bound[which] = 0;
  for (int i = tid; i < n; i += kLanes) keys[i] = a.keys[(long long)row * n + i];
  if (on && tid < 64) {
    const long long token = a.token_ids[row];
    const bool known = token >= 0 && token < a.vocab;
    const uint8_t* p = a.logits + row * a.row_stride + (known ? token : 0) * X::kBytes;
    const float x = TYPE == 2 ? *reinterpret_cast<const float*>(p)
                    : TYPE == 1 ? __builtin_bit_cast(float, (uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16)
                                : (float)*reinterpret_cast<const f16*>(p);
    Part own = {-__builtin_inff(), 0.f, 0.f, 0};
    if (tid < a.segments) own = parts[tid];
    const float most = wave_all(own.most, [](float p, float q) { return larger(p, q); });
    float rest = 0.f, weighted = 0.f, count = 0.f;
    if (own.most == most) {
      count = (float)own.count, rest = own.rest, weighted = own.weighted;
    } else if (own.most > -__builtin_inff()) {
      const float d = own.most - most, f = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f), z = (float)own.count + own.rest;
      rest = z * f;
      weighted = __builtin_fmaf(z, d, own.weighted) * f;
    }
    const auto add = [](float p, float q) { return p + q; };
    rest = wave_all(rest, add), weighted = wave_all(weighted, add), count = wave_all(count, add);
    double log_z = __builtin_nan(""), entropy = __builtin_nan("");
    if (__builtin_isfinite(most)) finish(count, rest, weighted, log_z, entropy);
    if (tid == 0) {
      shared_log_z[which] = log_z;
      shared_most[which] = most;
      a.logprob[row] = known ? (float)((double)(x - most) - log_z) : __builtin_nanf("");
      a.entropy[row] = (float)entropy;
    }
  }
  __syncthreads();
  // Of many keys: the first ones of each segment, `top` in all or a few more, bound the top'th key of the row from below;
  // what is not below the bound, little more than `top`, is ranked.
  const bool many = a.segments * a.top > (ROWS == 1 ? 128 : 32);
  const int leading = (a.top + a.segments - 1) / a.segments, m = on && many ? leading * a.segments : 0;
  for (int i = tid; i < m; i += kLanes) {
    const u64 key = keys[i / leading * a.top + i % leading];
    int ahead = 0;
#pragma unroll 8
    for (int j = 0; j < a.segments; ++j)
      for (int r = 0; r < leading; ++r) ahead += keys[j * a.top + r] > key;
    if (ahead == a.top - 1 && key) bound[which] = key;
  }
  if (many) {
    __syncthreads();
    const u64 border = bound[which];
    for (int i = tid; i < n; i += kLanes) {
      const u64 key = keys[i];
      if (key && key >= border) {
        const int at = atomicAdd(&n_ranked[which], 1);
        if (at < kRanked) ranked[which][at] = key;
      }
    }
    __syncthreads();
  }
  const bool fits = many && n_ranked[which] <= kRanked;
  const u64* from = fits ? ranked[which] : keys;
  const int count = fits ? n_ranked[which] : n;
  for (int i = tid; i < count; i += kLanes) {
    const u64 key = from[i];
    if (key == 0) continue;  // of a segment with fewer elements than ranks
    int ahead = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) ahead += from[j] > key;
    if (ahead < a.top) {
      a.top_ids[(long long)row * a.top + ahead] = index_of(key);
      a.top_logprobs[(long long)row * a.top + ahead] =
          (float)((double)(unordered((uint32_t)(key >> 32)) - shared_most[which]) - shared_log_z[which]);
    }
  }
}

// A lane holds 32 elements; the first 16 bytes of a segment may hold 7 (3) elements in front of it.  A workgroup of
// 1024 lanes takes a row of up to 32760 tokens alone, one of 512 half of that, which is one launch instead of two; where
// there are enough rows to fill the chip, segments of 256 lanes do more, since a CU runs several (one loads while another
// sums): 4096 x 32000 fp32 with 20 alternatives 105 us against 154, 4096 x 16000 bf16 56 against 61 with 512 lanes; but
// 300 x 9000 bf16 11.1 against 9.2, 200 x 30000 12.1 against 8.7 with 1024.
struct Plan {
  int threads, segments, segment;
};
Plan plan(int rows, int vocab, int type) {
  const int spare = type == 2 ? 3 : 7;
  Plan p;
  p.threads = 256;
  if (vocab + spare > 256 * 32) {
    if (vocab + spare <= 512 * 32 && rows <= 4 * kFewRows)
      p.threads = 512;
    else if (vocab > 16 * (256 * 32 - 8) || (vocab + spare <= 1024 * 32 && rows <= kFewRows))
      p.threads = 1024;
  }
  const int most = p.threads * 32 - 8;
  if (vocab + spare <= p.threads * 32) {
    p.segments = 1, p.segment = vocab;
  } else {
    p.segments = (vocab + most - 1) / most;
    p.segment = ((vocab + p.segments - 1) / p.segments + 7) / 8 * 8;
    p.segments = (vocab + p.segment - 1) / p.segment;
  }
  return p;
}

template <int TYPE>
int launch(const Args& a, int rows, int threads, hipStream_t s) {
  constexpr int kAll = 32 / Logits<TYPE>::kEach;
  const dim3 grid((unsigned)rows * (unsigned)a.segments);
  if (threads == 256)
    hipLaunchKernelGGL((logprobs_kernel<TYPE, 256, kAll>), grid, dim3(256), 0, s, a);
  else if (threads == 512)
    hipLaunchKernelGGL((logprobs_kernel<TYPE, 512, kAll>), grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((logprobs_kernel<TYPE, 1024, kAll>), grid, dim3(1024), 0, s, a);
  if (a.segments > 1) {
    const int rc = serving_after_launch();
    if (rc != SERVING_OK) return rc;
    if (a.segments * a.top <= 128 && rows >= 1024)
      hipLaunchKernelGGL((join_kernel<TYPE, 4>), dim3((unsigned)((rows + 3LL) / 4)), dim3(256), 0, s, a, rows);
    else
      hipLaunchKernelGGL((join_kernel<TYPE, 1>), dim3((unsigned)rows), dim3(256), 0, s, a, rows);
  }
  return serving_after_launch();
}

bool sizes_ok(int rows, int vocab, int top, int type) {
  return rows > 0 && vocab > 0 && vocab <= kMaxVocab && top >= 0 && top <= kMaxTop && top <= vocab && type >= 0 && type <= 2;
}

}  // namespace

extern "C" size_t serving_token_logprobs_workspace_bytes(int rows, int vocab, int top, int type) {
  if (!sizes_ok(rows, vocab, top, type)) return 0;
  const Plan p = plan(rows, vocab, type);
  if (p.segments == 1) return 0;
  return (size_t)rows * p.segments * (sizeof(Part) + (size_t)top * sizeof(u64));
}

extern "C" int serving_token_logprobs(const void* logits, long long row_stride, const int64_t* token_ids, float* logprob,
                                      float* entropy, int64_t* top_ids, float* top_logprobs, int rows, int vocab, int top,
                                      int type, void* workspace, size_t workspace_bytes, void* stream) {
  if (!logits || !token_ids || !logprob || !entropy || (top > 0 && (!top_ids || !top_logprobs))) return SERVING_E_NULL;
  if (!sizes_ok(rows, vocab, top, type)) return SERVING_E_SHAPE;
  const int bytes = type == 2 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % bytes) return SERVING_E_ALIGN;
  const Plan p = plan(rows, vocab, type);
  if ((long long)rows * p.segments * p.threads > 0xffffffffLL) return SERVING_E_TOO_LARGE;
  const size_t need = serving_token_logprobs_workspace_bytes(rows, vocab, top, type);
  if (need && (!workspace || workspace_bytes < need)) return SERVING_E_WORKSPACE;
  if (need && !aligned16(workspace)) return SERVING_E_ALIGN;
  Args a{static_cast<const uint8_t*>(logits), row_stride * bytes, token_ids, logprob, entropy, top_ids, top_logprobs,
         static_cast<Part*>(workspace), nullptr, vocab, top, p.segments, p.segment};
  if (need) a.keys = reinterpret_cast<u64*>(a.parts + (size_t)rows * p.segments);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (type == 0) return launch<0>(a, rows, p.threads, s);
  if (type == 1) return launch<1>(a, rows, p.threads, s);
  return launch<2>(a, rows, p.threads, s);
}
