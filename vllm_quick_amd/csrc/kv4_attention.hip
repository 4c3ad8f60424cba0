// Attention over the 4-bit paged cache: one pass over the keys and values with the running maximum and sum of the
// softmax, on 16x16x32 matrix instructions.
//
// Codes reach the matrix cores without being converted.  A code n in the low bits of a 16-bit lane IS the fp16 number
// n 2^-24 (a subnormal; four bits further up 16 n 2^-24), and the matrix instructions take subnormals exactly.  So a
// word of 8 codes becomes a fragment of 8 fp16 numbers with four ands and a shift, and the scales and leasts of the
// format stay outside the product:
//   q . k_j  =  scale_j (q . code_j) + least_j sum(q)             sum(q) once for each query
//   o        =  sum_j (p_j vscale_j) code_j + sum_j p_j vleast_j    the second sum is one number for all of a head's
//                                                                elements
// Where the sixteens stand in the keys' fragments the queries are divided by 16; in the values' they belong to whole
// rows of the result.
//
// A wave works on 16 NC columns (queries x heads of one kv head) and 32 keys at a time:
//   S^T = K Q^T   A = codes of 16 keys (lane & 15) x 32 elements, one 16-byte load a lane for a whole head of 128
//   O^T = V^T P^T  the result of the first product is, lane for lane, the B operand of the second: a lane's keys are
//                  4 g + 0..3 (g = lane >> 4) of both groups of 16; the format keeps the values of 16 tokens piece by
//                  piece, so that the same 4 keys of a piece are again one 16-byte load, and one byte permutation a
//                  word pairs the codes of neighbouring keys.
// Roundings: queries enter exactly (scaled by a power of two into fp16's range), w_j = p_j vscale_j is rounded to fp16
// once, all sums are fp32.  A code stands for zero at n_j = -least_j / vscale_j, not at 0, so w_j's rounding costs
// (n - n_j) + n_j steps of it; the second part, w_j's error times n_j, is the same for all elements and goes into the
// second sum (n_j to an eighth).  Only for fp16 results: bf16 ones are rounded coarser than what it repairs.
#include "kv4_cache.h"

namespace {

using namespace serving;

constexpr float kNone = -1e30f;  // below every score, yet finite: differences of it are numbers
constexpr int kTile = 32;        // keys of a step
constexpr float kSlack = 8.f;     // a probability may stand this many powers of two above 1 before the maximum moves
constexpr float kWeight = 0x1p7f;  // p vscale / (power of two above vscale) times this is rounded to fp16: below 2^15

struct AttendArgs {
  const void* query;
  long long q_token, q_head;
  const uint8_t* cache;
  const int32_t* tables;
  long long table_stride;
  const int32_t *seq_lens, *query_start;
  void* out;
  float* part_o;   // [tokens][heads][splits][D], sums of p v
  float* part_ml;  // [tokens][heads][splits][2], maximum (in powers of two) and sum of p
  int table_width, tokens, seqs, heads, kv_heads, group;
  int num_blocks, block_size;
  uint32_t per_block_magic;  // ceil(2^32 / (block_size / 16)), or 0 for blocks of 16
  float scale;               // of the scores, times log2(e)
  int window, max_query_len, splits;
};

// Uniform integers that no kernel here writes, through the scalar cache: a vector load would return behind all the
// loads of keys that were issued before it.
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ __forceinline__ scalar_ints scalar(const int32_t* p) { return (scalar_ints)(uintptr_t)p; }
__device__ __forceinline__ f16x2 as_pair(uint32_t w) { return __builtin_bit_cast(f16x2, w); }  // scale, least
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// 1 / v to an eighth of it, from the number's bits: the line of slope -1 through (log2 v, log2 1/v) that is nearest.
__device__ __forceinline__ float rough_reciprocal(float v) {
  return __builtin_bit_cast(float, 0x7ef311c7u - __builtin_bit_cast(uint32_t, v));
}
__device__ __forceinline__ float over_groups_max(float v) {  // of the four groups of 16 lanes
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Keeps a branch that is rarely taken a branch.
__device__ __forceinline__ void stay() { asm volatile(""); }

// One sequence as a wave sees it.
struct Sequence {
  int length;  // tokens in the cache
  int row;     // of its first query
  int queries;
  int before;  // length - queries: the position of its first query
};
__device__ __forceinline__ Sequence sequence(const AttendArgs& a, int b) {
  Sequence s;
  const long long most = (long long)a.table_width * a.block_size;
  s.length = max(0, (int)min((long long)scalar(a.seq_lens)[b], most));
  s.row = a.query_start ? scalar(a.query_start)[b] : b;
  s.queries = a.query_start ? scalar(a.query_start)[b + 1] - s.row : 1;
  if (s.row < 0 || s.row > a.tokens) s.row = a.tokens;
  s.queries = max(0, min(s.queries, a.tokens - s.row));
  s.before = s.length - s.queries;
  return s;
}

template <typename T, int D, int NC>
struct Wave {
  static constexpr int kSteps = D / 32;  // matrix instructions of 16 keys against 16 columns
  static constexpr int kRows = D / 16;   // tiles of 16 elements of the result
  static constexpr bool kRepair = __is_same(T, f16);

  const AttendArgs& a;
  const int c, g;
  // the step's keys, values and parameters; each is overwritten by the next step's as soon as it is used
  uint32_t k[2][kSteps];
  u32x4 v[2], kp[2], vp[2];
  f16x8 q[NC][kSteps];
  float qs[NC], al[NC];  // sum of the query, and what makes a score (in powers of two) of a product
  int lim[NC], low[NC];  // keys that a column sees: low .. lim - 1
  float shift[NC];       // p = 2^(al u + shift): no p passes 2^kSlack
  float sum[NC], flat[NC];
  f32x4 o[NC][kRows];
  float vref;                // power of two above every vscale so far
  const uint8_t* head_base;  // of this kv head in block 0
  scalar_ints table;
  long long block_bytes;
  int last_page;
  const uint8_t* base[2];  // where the next step's two groups of 16 tokens are
  int place[2];
  bool known[2];

  __device__ __forceinline__ Wave(const AttendArgs& args) : a(args), c(threadIdx.x & 15), g((threadIdx.x & 63) >> 4) {}

  __device__ __forceinline__ void begin(const Sequence& s, int b, int kv, int col0, int cols) {
    head_base = a.cache + (long long)kv * Kv4<D>::block_bytes(a.block_size);
    block_bytes = Kv4<D>::block_bytes(a.block_size) * a.kv_heads;
    table = scalar(a.tables + b * a.table_stride);
    last_page = max(0, page_of((s.length - 1) >> 4));
    vref = 0x1p-40f;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int col = col0 + 16 * n + c;
      const bool on = col < cols;
      const int qi = on ? col / a.group : 0, h = on ? col - qi * a.group : 0;
      lim[n] = on ? max(0, min(s.length, s.before + qi + 1)) : 0;
      low[n] = a.window > 0 ? max(0, lim[n] - a.window) : 0;
      const T* src = static_cast<const T*>(a.query) + (long long)(s.row + qi) * a.q_token + (kv * a.group + h) * a.q_head;
      typedef T vec8 __attribute__((ext_vector_type(8)));
      float x[kSteps][8], big = 0.f, total = 0.f;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        vec8 w = {};
        if (on) w = *reinterpret_cast<const vec8*>(src + (D / 4) * g + 8 * j);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[j][i] = (float)w[i];
          big = fmaxf(big, fabsf(x[j][i]));
          total += x[j][i];
        }
      }
      big = over_groups_max(big);
      total = over_groups_sum(total);
      // into [2^13, 2^14): a sixteenth of it, and of what is far below it, is still a normal fp16 number
      const int e = 14 - __builtin_amdgcn_frexp_expf(big);
      const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // element (i % 2) * 4 + i / 2 of the word is where the masks leave it
          const int el = (i & 1) * 4 + (i >> 1);
          q[n][j][i] = (f16)__builtin_ldexpf(sign * x[j][el], (i >> 1) & 1 ? e - 4 : e);
        }
      }
      qs[n] = __builtin_ldexpf(sign * total, e - 24);
      al[n] = __builtin_ldexpf(fabsf(a.scale), 24 - e);
      shift[n] = -kNone;
      sum[n] = flat[n] = 0.f;
#pragma unroll
      for (int m = 0; m < kRows; ++m) o[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  __device__ __forceinline__ int page_of(int sixteenth) const {
    return a.per_block_magic ? (int)__umulhi((uint32_t)max(0, sixteenth), a.per_block_magic) : max(0, sixteenth);
  }

  // The block that holds 16 tokens (behind the last page: the last one, whose tokens there are hidden).
  __device__ __forceinline__ int block_of(int sixteenth) const { return table[min(page_of(sixteenth), last_page)]; }

  __device__ __forceinline__ void aim(int tile, int block0, int block1) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int sixteenth = 2 * tile + s, block = s ? block1 : block0;
      known[s] = (uint32_t)block < (uint32_t)a.num_blocks;
      const int page = page_of(sixteenth);
      place[s] = page <= last_page ? 16 * sixteenth - page * a.block_size : 0;
      base[s] = head_base + (known[s] ? block : 0) * block_bytes;
    }
  }

  __device__ __forceinline__ void load_keys() {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* at = base[s] + (uint32_t)(place[s] * Kv4<D>::kTokenBytes) + (uint32_t)(c * Kv4<D>::kTokenBytes + g * (D / 8));
      if (D == 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) k[s][j] = w[j];
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(at);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) k[s][j] = w[j];
      }
    }
  }

  __device__ __forceinline__ void load_params() {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t at = (uint32_t)(Kv4<D>::key_params(a.block_size) + 4 * place[s]);
      kp[s] = *reinterpret_cast<const u32x4*>(base[s] + at + (uint32_t)(16 * g));
      vp[s] = *reinterpret_cast<const u32x4*>(base[s] + (at + 4 * (uint32_t)a.block_size) + (uint32_t)(16 * g));
      if (!known[s])  // a block that the cache does not have: its keys are NaN
        kp[s] = u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
    }
  }

  __device__ __forceinline__ void load_values() {
    const int piece = D == 128 ? c : c >> 1;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      v[s] = *reinterpret_cast<const u32x4*>(base[s] + (uint32_t)(Kv4<D>::values(a.block_size) + (place[s] / 16) * Kv4<D>::kGroupBytes) +
                                             (uint32_t)(piece * Kv4<D>::kPieceBytes + 16 * g));
  }

  __device__ __forceinline__ bool sees(int n, int from, int i) const {
    const int key = from + 16 * (i / 4) + 4 * g + i % 4;
    return key >= low[n] && key < lim[n];
  }

  // Scores of 32 keys to weights, the B operand of the second product.
  template <bool MASK>
  __device__ __forceinline__ void weigh(const f32x4 (&s)[2], int n, int from, float vinv, f16x8& p) {
    float u[8], e[8], w[8], least[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16x2 par = as_pair(kp[i / 4][i % 4]);
      u[i] = __builtin_fmaf(s[i / 4][i % 4], (float)par.x, (float)par.y * qs[n]);
    }
    if (MASK) {
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = sees(n, from, i) ? u[i] : kNone;
    }
    float most = u[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = fmaxf(most, u[i]);
    if (__any(__builtin_fmaf(al[n], most, shift[n]) > kSlack)) {
      stay();
      most = over_groups_max(most);  // (a column moves for its own keys only, whatever the wave's others do)
      const float next = __builtin_fmaf(al[n], most, shift[n]) > kSlack ? -al[n] * most : shift[n];
      const float f = exp2_(next - shift[n]);
      shift[n] = next;
      sum[n] *= f;
      flat[n] *= f;
#pragma unroll
      for (int m = 0; m < kRows; ++m) o[n][m] *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16x2 par = as_pair(vp[i / 4][i % 4]);
      e[i] = exp2_(__builtin_fmaf(al[n], u[i], shift[n]));
      w[i] = e[i] * ((float)par.x * vinv);
      least[i] = (float)par.y;
    }
    if (MASK) {  // (not 0 times what a hidden key's parameters may be)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool on = sees(n, from, i);
        e[i] = on ? e[i] : 0.f;
        w[i] = on ? w[i] : 0.f;
        least[i] = on ? least[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum[n] += e[i];
      flat[n] = __builtin_fmaf(e[i], least[i], flat[n]);
      p[i] = (f16)w[i];
      if (kRepair) {
        const float vs = (float)as_pair(vp[i / 4][i % 4]).x * vinv;
        flat[n] = __builtin_fmaf((float)p[i] - w[i], least[i] * rough_reciprocal(fmaxf(vs, 0x1p-40f)), flat[n]);
      }
    }
  }

  // 32 keys.  What the running maximum and the values' scales are measured against moves only when a probability would
  // pass 2^kSlack, or a scale its reference, which no step but the first few does: the four groups of lanes need to
  // agree on neither until then.
  template <bool MASK>
  __device__ __forceinline__ void step(int from, int length) {
    f32x4 s[NC][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const uint32_t w = k[h][j], x = w >> 8;
        const u32x4 f = {w & 0x000f000fu, w & 0x00f000f0u, x & 0x000f000fu, x & 0x00f000f0u};
#pragma unroll
        for (int n = 0; n < NC; ++n)
          s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, f), q[n][j],
                                                           j ? s[n][h] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      }
    }
    load_keys();
    if (MASK) {  // parameters behind the sequence may be anything
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (from + 16 * (i / 4) + 4 * g + i % 4 >= length) vp[i / 4][i % 4] = 0;
    }
    f16x2 big = as_pair(vp[0][0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) big = __builtin_elementwise_max(big, as_pair(vp[i / 4][i % 4]));
    if (__any((float)big.x >= vref)) {
      stay();
      const float ref = over_groups_max((float)big.x);
      const float next = fmaxf(vref, __builtin_ldexpf(1.f, __builtin_amdgcn_frexp_expf(ref)));
      const float f = vref * __builtin_amdgcn_rcpf(next);  // (of a power of two: exact)
      vref = next;
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int m = 0; m < kRows; ++m) o[n][m] *= f;
    }
    const float vinv = kWeight * __builtin_amdgcn_rcpf(vref);
    f16x8 p[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) weigh<MASK>(s[n], n, from, vinv, p[n]);
    load_params();
    // pairs of neighbouring keys side by side: 16 bits (4 elements) of each in one word
#pragma unroll
    for (int half = 0; half < (D == 128 ? 2 : 1); ++half) {
      const uint32_t pick = (D == 128 ? half : c & 1) ? 0x07060302u : 0x05040100u;
      u32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_perm(v[i / 2][2 * (i % 2) + 1], v[i / 2][2 * (i % 2)], pick);
      const u32x4 y = x >> 8;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32x4 f = (e & 2 ? y : x) & (e & 1 ? 0x00f000f0u : 0x000f000fu);
        const int m = 4 * half + e;
#pragma unroll
        for (int n = 0; n < NC; ++n)
          o[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, f), p[n], o[n][m], 0, 0, 0);
      }
    }
    load_values();
  }

  // Runs over tiles first, first + stride, .. < last; all columns see all of the tiles that lie in whole_from ..
  // whole_to - 1 of the keys.
  __device__ __forceinline__ void run(int first, int last, int stride, int length, int whole_from, int whole_to) {
    if (first >= last) return;
    aim(first, block_of(2 * first), block_of(2 * first + 1));
    load_keys();
    load_params();
    load_values();
    int next = min(first + stride, last - 1);  // (the last step loads some tile again, which nobody looks at)
    int b0 = block_of(2 * next), b1 = block_of(2 * next + 1);
    const auto advance = [&] {
      aim(next, b0, b1);
      next = min(next + stride, last - 1);
      b0 = block_of(2 * next), b1 = block_of(2 * next + 1);
    };
    const int whole_first = (whole_from + kTile - 1) / kTile, whole_last = min(last, whole_to / kTile);
    int i = first;
    while (true) {
      if (i >= whole_first)
        for (; i < whole_last; i += stride) {
          advance();
          step<false>(i * kTile, length);
        }
      if (i >= last) break;
      advance();
      step<true>(i * kTile, length);
      i += stride;
      if (i >= last) break;
    }
  }

  // Element d of the result of this lane's column, as sums of p v: out(piece of kEach elements, first element, values).
  template <typename F>
  __device__ __forceinline__ void results(int n, F&& out) {
    constexpr int kEach = kRows;  // neighbouring elements that a lane holds: element kEach (4 g + r) + m
    const float unit = vref * (0x1p24f / kWeight), rest = over_groups_sum(flat[n]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x[kEach];
#pragma unroll
      for (int m = 0; m < kEach; ++m) x[m] = __builtin_fmaf(o[n][m][r], m & 1 ? unit * 0.0625f : unit, rest);
      out(kEach * (4 * g + r), x);
    }
  }
};

// The rows of a sequence past max_query_len were promised not to exist: they say so.
template <typename T, int D>
__device__ void refuse_rows(const AttendArgs& a, const Sequence& s, int kv) {
  const int per_row = a.group * D;
  for (int qi = a.max_query_len; qi < s.queries; ++qi) {
    T* dst = static_cast<T*>(a.out) + ((long long)(s.row + qi) * a.heads + kv * a.group) * D;
    for (int i = threadIdx.x; i < per_row; i += blockDim.x) dst[i] = (T)__builtin_nanf("");
  }
}

// Few queries a sequence: a workgroup of four waves shares the keys of one column tile (or of one of `splits` pieces
// of them), joined through LDS; pieces are joined by a second kernel.
template <typename T, int D, int NC>
__global__ void __launch_bounds__(256, NC == 1 ? 3 : 2) attend_split_kernel(AttendArgs a) {
  constexpr int kCols = 16 * NC;
  __shared__ float part[4][kCols][D + 4];
  __shared__ float maxima[4][kCols], sums[4][kCols];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = blockIdx.x, b = pair / a.kv_heads, kv = pair - b * a.kv_heads;
  const int split = blockIdx.y, tile = blockIdx.z;
  const Sequence s = sequence(a, b);
  const int queries = min(s.queries, a.max_query_len), cols = queries * a.group;
  if (tile == 0 && split == 0 && queries < s.queries) refuse_rows<T, D>(a, s, kv);
  const int col0 = tile * kCols;
  if (col0 >= cols) return;
  Wave<T, D, NC> w(a);
  w.begin(s, b, kv, col0, cols);
  const int first_q = col0 / a.group, last_q = min(cols - 1, col0 + kCols - 1) / a.group;
  const int end = max(0, s.before + last_q + 1);            // keys that any column sees end here
  const int least_lim = max(0, s.before + first_q + 1);     // and those that all see, here
  const int start = a.window > 0 ? max(0, least_lim - a.window) : 0;
  const int most_low = a.window > 0 ? max(0, end - a.window) : 0;
  const int first_tile = start / kTile, tiles = (end + kTile - 1) / kTile - first_tile;
  const int t0 = first_tile + (int)((long long)max(0, tiles) * split / a.splits);
  const int t1 = first_tile + (int)((long long)max(0, tiles) * (split + 1) / a.splits);
  // (padding columns see nothing: a step that holds some is masked throughout only where the others are)
  w.run(t0 + wave, t1, 4, s.length, most_low, least_lim);

  const int c = w.c;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    w.results(n, [&](int d, const float* x) {
#pragma unroll
      for (int m = 0; m < D / 16; m += 4)
        *reinterpret_cast<f32x4*>(&part[wave][16 * n + c][d + m]) = f32x4{x[m], x[m + 1], x[m + 2], x[m + 3]};
    });
    const float total = over_groups_sum(w.sum[n]);
    if (w.g == 0) {
      maxima[wave][16 * n + c] = fmaxf(-w.shift[n], -1e38f);  // (finite, whatever the query's size)
      sums[wave][16 * n + c] = total;
    }
  }
  __syncthreads();
  constexpr int kEach = D * kCols / 256;  // elements of a column that a thread joins
  constexpr int kPer = D / kEach;
  const int col = threadIdx.x / kPer, d0 = (threadIdx.x % kPer) * kEach;
  if (col0 + col >= cols) return;
  float top = maxima[0][col];
#pragma unroll
  for (int i = 1; i < 4; ++i) top = fmaxf(top, maxima[i][col]);
  float total = 0.f, x[kEach] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = exp2_(maxima[i][col] - top);
    total = __builtin_fmaf(sums[i][col], f, total);
#pragma unroll
    for (int d = 0; d < kEach; ++d) x[d] = __builtin_fmaf(part[i][col][d0 + d], f, x[d]);
  }
  const int qi = (col0 + col) / a.group, head = kv * a.group + (col0 + col) - qi * a.group;
  const long long at = (long long)(s.row + qi) * a.heads + head;
  if (a.splits == 1) {
    const float inv = total == 0.f ? 0.f : 1.f / total;
    T* dst = static_cast<T*>(a.out) + at * D + d0;
#pragma unroll
    for (int d = 0; d < kEach; ++d) dst[d] = (T)(total == 0.f ? 0.f : x[d] * inv);
  } else {
    float* dst = a.part_o + (at * a.splits + split) * D + d0;
#pragma unroll
    for (int d = 0; d < kEach; ++d) dst[d] = x[d];
    if (d0 == 0) {
      float* ml = a.part_ml + (at * a.splits + split) * 2;
      ml[0] = top;
      ml[1] = total;
    }
  }
}

// Joins the pieces of a query head: one wave each.
template <typename T, int D>
__global__ void __launch_bounds__(256) attend_join_kernel(AttendArgs a) {
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= (long long)a.tokens * a.heads) return;
  const int row = (int)(at / a.heads);
  if (a.query_start) {  // rows of no sequence stay as they are, rows past max_query_len too: the first kernel wrote them
    int lo = 0, hi = a.seqs;  // the last sequence that begins at or before this row
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.query_start[mid] <= row)
        lo = mid;
      else
        hi = mid;
    }
    if (row < a.query_start[lo] || row >= min(a.query_start[lo + 1], a.query_start[lo] + a.max_query_len)) return;
  }
  const int lane = threadIdx.x & 63;
  const float* ml = a.part_ml + at * a.splits * 2;
  float top = -1e38f;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[2 * s]);
  float total = 0.f, x[D / 64] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float f = exp2_(ml[2 * s] - top);
    total = __builtin_fmaf(ml[2 * s + 1], f, total);
    const float* src = a.part_o + (at * a.splits + s) * D + lane * (D / 64);
#pragma unroll
    for (int d = 0; d < D / 64; ++d) x[d] = __builtin_fmaf(src[d], f, x[d]);
  }
  T* dst = static_cast<T*>(a.out) + at * D + lane * (D / 64);
#pragma unroll
  for (int d = 0; d < D / 64; ++d) dst[d] = (T)(total == 0.f ? 0.f : x[d] / total);
}

// Many queries a sequence: each wave has columns of its own and runs over all the keys that they see; the four waves of
// a workgroup hold neighbouring columns, so that they read the same keys at about the same time.
template <typename T, int D, int NC>
__global__ void __launch_bounds__(256, 2) attend_prompt_kernel(AttendArgs a) {
  constexpr int kCols = 16 * NC;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = blockIdx.x, b = pair / a.kv_heads, kv = pair - b * a.kv_heads;
  const Sequence s = sequence(a, b);
  const int queries = min(s.queries, a.max_query_len), cols = queries * a.group;
  if (blockIdx.y == 0 && queries < s.queries) refuse_rows<T, D>(a, s, kv);
  const int group_cols = 4 * kCols, groups = (cols + group_cols - 1) / group_cols;
  if ((int)blockIdx.y >= groups) return;
  // the columns that see most come first: what is left at the end is short
  const int col0 = (groups - 1 - (int)blockIdx.y) * group_cols + wave * kCols;
  if (col0 >= cols) return;
  Wave<T, D, NC> w(a);
  w.begin(s, b, kv, col0, cols);
  const int first_q = col0 / a.group, last_q = min(cols - 1, col0 + kCols - 1) / a.group;
  const int end = max(0, s.before + last_q + 1), least_lim = max(0, s.before + first_q + 1);
  const int start = a.window > 0 ? max(0, least_lim - a.window) : 0;
  const int most_low = a.window > 0 ? max(0, end - a.window) : 0;
  w.run(start / kTile, (end + kTile - 1) / kTile, 1, s.length, most_low, least_lim);
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const float total = over_groups_sum(w.sum[n]);
    const int col = col0 + 16 * n + w.c;
    const int qi = col / a.group, head = kv * a.group + col - qi * a.group;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    w.results(n, [&](int d, const float* x) {
      if (col >= cols) return;
      typedef T piece __attribute__((ext_vector_type(D / 16)));
      piece y;
#pragma unroll
      for (int m = 0; m < D / 16; ++m) y[m] = (T)(total == 0.f ? 0.f : x[m] * inv);
      *reinterpret_cast<piece*>(static_cast<T*>(a.out) + ((long long)(s.row + qi) * a.heads + head) * D + d) = y;
    });
  }
}

// How a call is laid over the chip, from its sizes alone.
struct Plan {
  bool prompt;
  int nc, tiles, splits;
};
Plan plan(int seqs, int heads, int kv_heads, int max_query_len, int max_seq_len, int window) {
  const long long cols = (long long)max_query_len * (heads / kv_heads);
  Plan p;
  p.prompt = cols > 64;
  p.nc = cols > 16 ? 2 : 1;
  p.tiles = (int)((cols + 16 * p.nc - 1) / (16 * p.nc));
  p.splits = 1;
  if (p.prompt) return p;
  const long long groups = (long long)seqs * kv_heads * p.tiles;
  long long keys = max_seq_len;
  if (window > 0 && window + max_query_len < keys) keys = window + max_query_len;
  const long long most = (keys + 511) / 512;  // four waves with four tiles each
  long long splits = (1024 + groups - 1) / groups;
  splits = splits < most ? splits : most;
  p.splits = (int)(splits < 1 ? 1 : splits > 256 ? 256 : splits);
  return p;
}

template <typename T, int D>
int launch(const AttendArgs& a, const Plan& p, hipStream_t s) {
  const unsigned pairs = (unsigned)a.seqs * (unsigned)a.kv_heads;
  if (p.prompt) {
    const dim3 grid(pairs, (unsigned)((p.tiles + 3) / 4));
    hipLaunchKernelGGL((attend_prompt_kernel<T, D, 2>), grid, dim3(256), 0, s, a);
    return serving_after_launch();
  }
  const dim3 grid(pairs, (unsigned)p.splits, (unsigned)p.tiles);
  if (p.nc == 1)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 1>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attend_split_kernel<T, D, 2>), grid, dim3(256), 0, s, a);
  int rc = serving_after_launch();
  if (rc != SERVING_OK || p.splits == 1) return rc;
  const long long rows = (long long)a.tokens * a.heads;
  hipLaunchKernelGGL((attend_join_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
  return serving_after_launch();
}

bool sizes_ok(int tokens, int seqs, int heads, int kv_heads, int max_query_len, int max_seq_len, int window) {
  return tokens > 0 && seqs > 0 && heads > 0 && heads <= 65535 && kv_heads > 0 && kv_heads <= heads && heads % kv_heads == 0 &&
         max_query_len > 0 && max_seq_len > 0 && max_seq_len <= (1 << 27) && window >= 0;
}

}  // namespace

extern "C" size_t serving_attend_kv4_workspace_bytes(int tokens, int seqs, int heads, int kv_heads, int head_size,
                                                     int max_query_len, int max_seq_len, int window) {
  if (!sizes_ok(tokens, seqs, heads, kv_heads, max_query_len, max_seq_len, window) || !head_size_ok(head_size)) return 0;
  const Plan p = plan(seqs, heads, kv_heads, max_query_len, max_seq_len, window);
  return p.splits == 1 ? 0 : (size_t)tokens * heads * p.splits * (head_size + 2) * sizeof(float);
}

extern "C" int serving_attend_kv4(const void* query, long long q_token, long long q_head, const void* cache,
                                  const int32_t* tables, long long table_stride, int table_width, const int32_t* seq_lens,
                                  const int32_t* query_start, void* out, int tokens, int seqs, int heads, int kv_heads,
                                  int head_size, long long num_blocks, int block_size, float scale, int window,
                                  int max_query_len, int max_seq_len, int bf16_in, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (!query || !cache || !tables || !seq_lens || !out) return SERVING_E_NULL;
  if (!head_size_ok(head_size)) return SERVING_E_HEAD;
  if (!block_size_ok(block_size)) return SERVING_E_BLOCK;
  if (!sizes_ok(tokens, seqs, heads, kv_heads, max_query_len, max_seq_len, window) || table_width <= 0 || table_stride < 0 ||
      num_blocks <= 0 || num_blocks > 0x7fffffffLL || (!query_start && tokens != seqs) || (!query_start && max_query_len != 1) ||
      !__builtin_isfinite(scale))
    return SERVING_E_SHAPE;
  if ((long long)table_width * block_size > (1LL << 27)) return SERVING_E_TOO_LARGE;
  if (!aligned16(query) || !aligned16(cache) || !aligned16(out) || q_token % 8 || q_head % 8) return SERVING_E_ALIGN;
  const Plan p = plan(seqs, heads, kv_heads, max_query_len, max_seq_len, window);
  const size_t need = serving_attend_kv4_workspace_bytes(tokens, seqs, heads, kv_heads, head_size, max_query_len, max_seq_len, window);
  if (need && (!workspace || workspace_bytes < need)) return SERVING_E_WORKSPACE;
  if (need && !aligned16(workspace)) return SERVING_E_ALIGN;
  if ((long long)seqs * kv_heads > 0x7fffffLL || p.tiles > 4 * 65535LL || (long long)tokens * heads > (1LL << 33))
    return SERVING_E_TOO_LARGE;
  const int sixteens = block_size / 16;
  AttendArgs a{query, q_token, q_head, static_cast<const uint8_t*>(cache), tables, table_stride, seq_lens, query_start, out,
               static_cast<float*>(workspace), nullptr, table_width, tokens, seqs, heads, kv_heads, heads / kv_heads,
               (int)num_blocks, block_size,
               sixteens == 1 ? 0u : (uint32_t)(((1ULL << 32) + sixteens - 1) / sixteens),
               scale * 1.44269504088896340736f, window, max_query_len, p.splits};
  if (need) a.part_ml = a.part_o + (size_t)tokens * heads * p.splits * head_size;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_size == 64) return bf16_in ? launch<bf16, 64>(a, p, s) : launch<f16, 64>(a, p, s);
  return bf16_in ? launch<bf16, 128>(a, p, s) : launch<f16, 128>(a, p, s);
}
