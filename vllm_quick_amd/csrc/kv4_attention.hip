// Attention over the 4-bit paged cache: one pass over the keys and values with the running maximum and sum of the
// softmax, on 16x16x32 matrix instructions.
//
// Codes reach the matrix cores without being converted.  A code n in the low bits of a 16-bit lane IS the fp16 number
// n 2^-24 (a subnormal; four bits further up 16 n 2^-24), which the matrix instructions take.  So a word of 8 codes
// becomes a fragment of 8 fp16 numbers with four ands and a shift, and the scales and leasts of the format stay outside
// the product:
//   q . k_j  =  scale_j (q . code_j) + least_j sum(q)             sum(q) once for each query
//   o        =  sum_j (p_j vscale_j) code_j + sum_j p_j vleast_j    the second sum is one number for all of a head's
//                                                                elements
// Where the sixteens stand in the keys' fragments the queries are divided by 16.  The values' codes all go in as 16 n
// (two shifts a word more): a product of n 2^-24 is cut off at some 2^-17 of it, always downwards, which in a long
// sequence, where the sum of w_j code_j is a hundred times the result, showed as 6e-4 of an fp16 result (26 000 keys);
// of 16 n 2^-24 a sixteenth of that is cut off.
//
// A wave works on 16 NC columns (queries x heads of one kv head) and 32 keys at a time:
//   S^T = K Q^T   A = codes of 16 keys (lane & 15) x 32 elements, one 16-byte load a lane for a whole head of 128
//   O^T = V^T P^T  the result of the first product is, lane for lane, the B operand of the second: a lane's keys are
//                  4 g + 0..3 (g = lane >> 4) of both groups of 16; the format keeps the values of 16 tokens piece by
//                  piece, so that the same 4 keys of a piece are again one 16-byte load, and one byte permutation a
//                  word pairs the codes of neighbouring keys.
// Roundings: queries enter exactly (scaled by a power of two into fp16's range), w_j = p_j vscale_j is rounded to fp16
// once, all sums are fp32.  What a rounding takes from w_j or adds to it, its code multiplies, by up to 15.  For fp16 results
//   o = sum_j w_j (code_j - zero_j) + sum_j p_j (vleast_j + zero_j vscale_j),
// with zero_j near the code that would stand for 0 (any number is right), and w_j zero_j taken off with the rounded w_j, in a
// matrix instruction of its own: a rounding then costs about its share of the value, and nothing that the sum of p_j or the
// second sum take depends on it, however small w_j is.  bf16 results are rounded coarser than that.  2 x 2048 queries of 64
// heads of 128 take 770 us so in fp16, some 40 less with 7.5 for every zero_j (and 1.4 times the error), 712 in bf16.
#include "kv4_cache.h"

namespace {

using namespace serving;

constexpr float kNone = -0x1p127f;  // below every score, yet finite: differences of it are numbers
constexpr int kTile = 32;        // keys of a step
constexpr int kRun = 32;         // steps between two settings aside
constexpr float kWeightLog = 7.f;      // what a column is held against is set so that no p vscale of a step passes 2^7,
constexpr float kMostWeight = 15.f;    // and again when one may pass 2^15, which fp16 holds
constexpr float kLeastScale = 0x1p-24f;  // of a token whose values are all alike, for that purpose: fp16's least number

// Scores beyond kFar have digits of 4 and more: a wave that is held against one rounds scores by themselves from then on,
// in steps that take 1.7 times as long.
constexpr float kFar = 0x1p25f;

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
  int window, max_query_len;
  int search;       // whether workgroups are numbered through all sequences, or each sequence has `tiles` of them
  int splits;       // pieces that a sequence is cut into at most
  int least;        // steps that a piece has at least, about,
  float per_piece;  // and what share of the steps of all sequences together, but for a sequence's rounding
};

// Uniform integers that no kernel here writes, through the scalar cache: a vector load would return behind all the
// loads of keys that were issued before it.
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ __forceinline__ scalar_ints scalar(const int32_t* p) { return (scalar_ints)(uintptr_t)p; }
__device__ __forceinline__ f16x2 as_pair(uint32_t w) { return __builtin_bit_cast(f16x2, w); }  // scale, least
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// least / scale of two keys within -15 .. 0, to an eighth of it where the scale is a normal number: 1 / scale from the
// number's bits, the line of slope -1 through (log2 v, log2 1/v) that is nearest.
__device__ __forceinline__ f16x2 minus_zero(uint32_t scales, f16x2 leasts) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const f16x2 z = leasts * __builtin_bit_cast(f16x2, u16x2{0x7798, 0x7798} - __builtin_bit_cast(u16x2, scales));
  return __builtin_elementwise_min(__builtin_elementwise_max(z, f16x2{(f16)-15.f, (f16)-15.f}), f16x2{(f16)0.f, (f16)0.f});
}
__device__ __forceinline__ float over_groups_max(float v) {  // of the four groups of 16 lanes
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Keeps what is worked out of x in a branch that is rarely taken out of the registers before it.
template <typename V>
__device__ __forceinline__ V here(V x) {
  asm volatile("" : "+v"(x));
  return x;
}

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

template <typename T, int D, int NC, bool ONCE>
struct Wave {
  static constexpr int kSteps = D / 32;  // matrix instructions of 16 keys against 16 columns
  static constexpr int kRows = D / 16;   // tiles of 16 elements of the result
  static constexpr bool kCentred = __is_same(T, f16);

  const AttendArgs& a;
  const int c, g;
  // the step's keys, values and parameters; each is overwritten by the next step's as soon as it is used
  uint32_t k[2][kSteps];
  u32x4 v[2], kp[2], vp[2];
  f16x8 q[NC][kSteps];
  float qs[NC];          // sum of the query, in the unit of the scores
  int lim[NC], low[NC];  // keys that a column sees: low .. lim - 1
  int least_low;         // of all columns of the wave
  float shift[NC];       // p = 2^(score + shift)
  float sum[NC], flat[NC];
  float unit_score[NC];  // what makes a score (in powers of two) of a product
  float* kept;                        // in LDS: [16 NC][D + 4], what was set aside of the sums of p v,
  float kept_sum[NC], kept_shift[NC];  // of p, and the shift that both go with
  bool keeps;
  bool far;  // some column is held against a score beyond kFar: steps are taken as those with masks, which see to that
  f32x4 o[NC][kRows], off[NC];  // sums of w code and, in each element, of w (- zero) (kCentred)
  const uint8_t* head_base;  // of this kv head in block 0
  scalar_ints table;
  long long block_bytes;
  int last_page;
  const uint8_t* base[2];  // where the next step's two groups of 16 tokens are
  int place[2];
  bool known[2], known_now[2];  // whether the cache has their blocks, and those of the keys in the registers

  __device__ __forceinline__ Wave(const AttendArgs& args) : a(args), c(threadIdx.x & 15), g((threadIdx.x & 63) >> 4) {}

  // Where the keys are, and the loads of the first tile.  No length is asked for: a tile behind the sequence loads what
  // some block of the table, or block 0, holds, and nobody looks at it.
  __device__ __forceinline__ void first_loads(int b, int kv, int first, float* lds) {
    kept = lds;
    keeps = far = false;
    head_base = a.cache + (long long)kv * Kv4<D>::block_bytes(a.block_size);
    block_bytes = Kv4<D>::block_bytes(a.block_size) * a.kv_heads;
    table = scalar(a.tables + b * a.table_stride);
    last_page = a.table_width - 1;
    aim(first, block_of(2 * first), block_of(2 * first + 1));
    load_keys();
    load_params();
    load_values();
  }

  // The queries.
  __device__ __forceinline__ void begin(const Sequence& s, int kv, int col0, int cols) {
    last_page = max(0, page_of((s.length - 1) >> 4));
    least_low = a.window > 0 ? max(0, s.before + col0 / a.group + 1 - a.window) : 0;
    float x[NC][kSteps][8], big[NC];
    const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int col = col0 + 16 * n + c;
      const bool on = col < cols;
      const int qi = on ? col / a.group : 0, h = on ? col - qi * a.group : 0;
      lim[n] = on ? max(0, min(s.length, s.before + qi + 1)) : 0;
      low[n] = a.window > 0 ? max(0, lim[n] - a.window) : 0;
      const T* src = static_cast<const T*>(a.query) + (long long)(s.row + qi) * a.q_token + (kv * a.group + h) * a.q_head;
      typedef T vec8 __attribute__((ext_vector_type(8)));
      float most = 0.f, total = 0.f;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        vec8 w = {};
        if (on) w = *reinterpret_cast<const vec8*>(src + (D / 4) * g + 8 * j);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[n][j][i] = sign * (float)w[i];
          most = fmaxf(most, fabsf(x[n][j][i]));
          total += x[n][j][i];
        }
      }
      qs[n] = over_groups_sum(total);
      big[n] = over_groups_max(most < __builtin_inff() ? most : 0.f);
    }
    // Each column by a power of two of its own, its largest element into [2^13, 2^14): a sixteenth of it, and of what is far
    // below it, is still a normal fp16 number, and what is not is 2^-38 of the column's largest score.
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int e = 14 - __builtin_amdgcn_frexp_expf(big[n]);
      unit_score[n] = __builtin_ldexpf(fabsf(a.scale), 24 - e);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // element (i % 2) * 4 + i / 2 of the word is where the masks leave it
          const int el = (i & 1) * 4 + (i >> 1);
          q[n][j][i] = (f16)__builtin_ldexpf(x[n][j][el], (i >> 1) & 1 ? e - 4 : e);
        }
      }
      qs[n] = __builtin_ldexpf(qs[n], e - 24) * unit_score[n];
      shift[n] = -kNone;
      sum[n] = flat[n] = 0.f;
#pragma unroll
      for (int m = 0; m < kRows; ++m) o[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
      off[n] = f32x4{0.f, 0.f, 0.f, 0.f};
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
      known_now[s] = known[s];
      known[s] = (uint32_t)block < (uint32_t)a.num_blocks;
      const int page = page_of(sixteenth);
      place[s] = page <= last_page ? 16 * sixteenth - page * a.block_size : 0;
      base[s] = head_base + (known[s] ? block : 0) * block_bytes;
    }
  }

  // Where each key is read once (ONCE: one column tile) the codes pass the caches by: 8 x 65536 keys 82 us against 91.
  // (The parameters of several tiles share a line.)
  template <typename V>
  static __device__ __forceinline__ V get(const uint8_t* at) {
    return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const V*>(at)) : *reinterpret_cast<const V*>(at);
  }

  __device__ __forceinline__ void load_keys() {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* at = base[s] + (uint32_t)(place[s] * Kv4<D>::kTokenBytes) + (uint32_t)(c * Kv4<D>::kTokenBytes + g * (D / 8));
      if (D == 128) {
        const u32x4 w = get<u32x4>(at);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) k[s][j] = w[j];
      } else {
        const u32x2 w = get<u32x2>(at);
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
    }
  }

  __device__ __forceinline__ void load_values() {
    const int piece = D == 128 ? c : c >> 1;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      v[s] = get<u32x4>(base[s] + (uint32_t)(Kv4<D>::values(a.block_size) + (place[s] / 16) * Kv4<D>::kGroupBytes) +
                        (uint32_t)(piece * Kv4<D>::kPieceBytes + 16 * g));
  }

  __device__ __forceinline__ bool sees(int n, int from, int i) const {
    const int key = from + 16 * (i / 4) + 4 * g + i % 4;
    return key >= low[n] && key < lim[n];
  }

  // Scores of 32 keys to weights, the B operand of the second product.  level: what the values' codes of zero stand for
  // (kCentred); limit: no p above 2^limit makes a p vscale of this lane pass 2^kMostWeight.
  template <bool MASK>
  __device__ __forceinline__ void weigh(const f32x4 (&s)[2], int n, int from, const float (&level)[8], float limit, f16x8& p) {
    float t[8], ks[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ks[i] = (float)as_pair(kp[i / 4][i % 4]).x * unit_score[n];
      if (MASK && !known_now[i / 4]) ks[i] = __builtin_nanf("");  // of a block that the cache does not have
    }
    const auto score = [&](int i, float more) {
      return __builtin_fmaf(ks[i], s[i / 4][i % 4], __builtin_fmaf((float)as_pair(kp[i / 4][i % 4]).y, qs[n], more));
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = MASK ? score(i, 0.f) + shift[n] : score(i, shift[n]);  // (a far score is rounded alike whatever is added)
      if (MASK) t[i] = sees(n, from, i) ? t[i] : kNone;
    }
    float most = t[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = fmaxf(most, t[i]);
    if (__any(most > limit)) {
      const auto log_scale = [&](int i) {
        return (float)__builtin_amdgcn_frexp_expf(fmaxf((float)as_pair(here(vp[i / 4][i % 4])).x, kLeastScale));
      };
      const auto heaviest = [&] {  // log2 of the largest p vscale, or a little above it
        float x = kNone;
#pragma unroll
        for (int i = 0; i < 8; ++i) x = fmaxf(x, t[i] + log_scale(i));
        return over_groups_max(x);
      };
      // (a column moves for its own keys only, whatever the wave's others do)
      float passed = kNone, top = kNone;  // of score + log2 vscale, or a little above it
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float more = log_scale(i);
        passed = fmaxf(passed, t[i] + more);
        if (!MASK) top = fmaxf(top, score(i, more));
      }
      const bool moves = over_groups_max(passed) > kMostWeight;
      bool aside = moves;
      float next = shift[n];
      if (!MASK) {
        top = over_groups_max(top);
        next = moves ? fminf(kWeightLog - top, next) : next;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = score(i, next);  // (rounded as outside, which other columns may have called for)
        aside = moves && (fabsf(top) >= kFar || fabsf(qs[n]) * 0x1p16f >= kFar);  // (a key's least value is below 2^16)
      }
      // A far score, or what a far score's parts have put aside of where it was to come: a score is rounded by itself then, so
      // that its difference to what it is held against is that of two scores.
      if (MASK || __any(aside)) {
        if (!MASK) aside = aside && !(fabsf(heaviest() - kWeightLog) <= 4.f && fabsf(next) < kFar);
        float peak = kNone;
        top = kNone;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (MASK && !sees(n, from, i)) continue;
          const float x = score(i, here(0.f));
          peak = fmaxf(peak, x);
          top = fmaxf(top, x + log_scale(i));
        }
        peak = over_groups_max(peak), top = over_groups_max(top);
        const bool beyond = fabsf(peak) >= kFar;
        next = aside ? fminf(beyond ? -peak : kWeightLog - top, shift[n]) : next;
        far |= __any(aside && (!MASK || beyond));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (MASK || aside) t[i] = score(i, here(0.f)) + next;
          if (MASK) t[i] = sees(n, from, i) ? t[i] : kNone;
        }
      }
      const float f = exp2_(next - shift[n]);
      shift[n] = next;
      sum[n] *= f;
      flat[n] *= f;
#pragma unroll
      for (int m = 0; m < kRows; ++m) o[n][m] *= f;
      off[n] *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16x2 par = as_pair(vp[i / 4][i % 4]);
      float e = exp2_(t[i]), w = e * (float)par.x, least = kCentred ? level[i] : (float)par.y;
      if (MASK) {  // (not 0 times what a hidden key's parameters may be)
        const bool on = sees(n, from, i);
        e = on ? e : 0.f;
        w = on ? w : 0.f;
        least = on ? least : 0.f;
      }
      p[i] = (f16)w;
      sum[n] += e;
      flat[n] = __builtin_fmaf(e, least, flat[n]);
    }
  }

  // 32 keys.  What a column is held against, the running maximum of p vscale over the keys that it sees, moves only when one
  // would pass 2^8 of it, which no step but the first few does: the four groups of lanes need not agree on it until then.
  // (The maximum of the product: a key of a large scale that is hardly attended to, or not seen, must not cost the others
  // their digits in fp16.)
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
    if (MASK) {  // parameters behind the sequence, before every window and of unknown blocks may be anything
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = from + 16 * (i / 4) + 4 * g + i % 4;
        if (key >= length || key < least_low || !known_now[i / 4]) vp[i / 4][i % 4] = 0;
      }
    }
    f16x2 big = as_pair(vp[0][0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) big = __builtin_elementwise_max(big, as_pair(vp[i / 4][i % 4]));
    const float limit = kMostWeight - (float)__builtin_amdgcn_frexp_expf(fmaxf((float)big.x, kLeastScale));
    f16x8 p[NC], zero;  // (zero: negative)
    float level[8];
    if (kCentred) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint32_t a0 = vp[i / 4][i % 4], a1 = vp[i / 4][i % 4 + 1];
        const f16x2 z = minus_zero(__builtin_amdgcn_perm(a1, a0, 0x05040100u), as_pair(__builtin_amdgcn_perm(a1, a0, 0x07060302u)));
        zero[i] = z.x, zero[i + 1] = z.y;
        level[i] = __builtin_fmaf((float)as_pair(a0).x, -(float)z.x, (float)as_pair(a0).y);
        level[i + 1] = __builtin_fmaf((float)as_pair(a1).x, -(float)z.y, (float)as_pair(a1).y);
      }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) weigh<MASK>(s[n], n, from, level, limit, p[n]);
    load_params();
    // pairs of neighbouring keys side by side: 16 bits (4 elements) of each in one word
#pragma unroll
    for (int half = 0; half < (D == 128 ? 2 : 1); ++half) {
      const uint32_t pick = (D == 128 ? half : c & 1) ? 0x07060302u : 0x05040100u;
      u32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_perm(v[i / 2][2 * (i % 2) + 1], v[i / 2][2 * (i % 2)], pick);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32x4 f = (e == 0 ? x << 4 : e == 1 ? x : e == 2 ? x >> 4 : x >> 8) & 0x00f000f0u;
        const int m = 4 * half + e;
#pragma unroll
        for (int n = 0; n < NC; ++n)
          o[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, f), p[n], o[n][m], 0, 0, 0);
      }
    }
    load_values();
    if (kCentred) {
#pragma unroll
      for (int n = 0; n < NC; ++n)
        off[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(zero, p[n], off[n], 0, 0, 0);
    }
  }

  // Runs over tiles first, first + stride, .. < last, the first of them loaded; all columns see all of the tiles that lie
  // in whole_from .. whole_to - 1 of the keys.
  // ALONE: a wave runs over all the keys by itself, which makes setting aside worth its place where scores are far too.
  template <bool ALONE>
  __device__ __forceinline__ void run(int first, int last, int stride, int length, int whole_from, int whole_to) {
    if (first >= last) return;
    int next = min(first + stride, last - 1);  // (the last step loads some tile again, which nobody looks at)
    int b0 = block_of(2 * next), b1 = block_of(2 * next + 1);
    const auto advance = [&] {
      aim(next, b0, b1);
      next = min(next + stride, last - 1);
      b0 = block_of(2 * next), b1 = block_of(2 * next + 1);
    };
    const int whole_first = (whole_from + kTile - 1) / kTile, whole_last = min(last, whole_to / kTile);
    int i = first, masked = 0;
    while (true) {
      if (i >= whole_first && !far) {
        const int stop = min(whole_last, i + kRun * stride);
        for (; i < stop && known[0] && known[1]; i += stride) {
          advance();
          step<false>(i * kTile, length);
        }
        if (i >= stop && i < whole_last) {
          set_aside();
          continue;
        }
      }
      if (i >= last) break;
      advance();
      step<true>(i * kTile, length);
      i += stride;
      if (i >= last) break;
      if (ALONE && far && ++masked % kRun == 0) set_aside();
    }
  }

  // Adds what the registers hold to what LDS keeps, and begins anew.  The codes are not centred, so that the two sums
  // that make a result are many times larger than it, the more so the longer the sequence: over 60 000 keys of one wave
  // fp16 results are 2.9e-4 off with this, 6.9e-4 without.  Each lane has places of its own: no barrier.
  __device__ __forceinline__ void set_aside() {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const float f = keeps ? exp2_(shift[n] - kept_shift[n]) : 0.f;
      kept_sum[n] = keeps ? __builtin_fmaf(kept_sum[n], f, sum[n]) : sum[n];
      kept_shift[n] = shift[n];
      results(n, [&](int d, const float* x) {
        f32x4* at = reinterpret_cast<f32x4*>(kept + (16 * n + c) * (D + 4) + d);
#pragma unroll
        for (int m = 0; m < kRows; m += 4) {
          f32x4 y = {x[m], x[m + 1], x[m + 2], x[m + 3]};
          if (keeps) y += at[m / 4] * f;
          at[m / 4] = y;
        }
      });
      sum[n] = flat[n] = 0.f;
#pragma unroll
      for (int m = 0; m < kRows; ++m) o[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
      off[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    keeps = true;
  }

  // Element d of the result of this lane's column, as sums of p v: out(first of kEach elements, values).
  template <typename F>
  __device__ __forceinline__ void results(int n, F&& out) {
    constexpr int kEach = kRows;  // neighbouring elements that a lane holds: element kEach (4 g + r) + m
    const float rest = kCentred ? over_groups_sum(flat[n]) + off[n][0] : over_groups_sum(flat[n]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x[kEach];
#pragma unroll
      for (int m = 0; m < kEach; ++m) x[m] = __builtin_fmaf(o[n][m][r], 0x1p20f, rest);
      out(kEach * (4 * g + r), x);
    }
  }
};

// Keys that columns first .. last of a tile see (some of them: tiles first_tile .. last_tile - 1; all: keys whole_from
// .. whole_to - 1).
struct Range {
  int first_tile, last_tile, whole_from, whole_to;
};
__device__ __forceinline__ Range range(const AttendArgs& a, const Sequence& s, int first, int last) {
  const int end = max(0, s.before + last / a.group + 1), whole_to = max(0, s.before + first / a.group + 1);
  const int start = a.window > 0 ? max(0, whole_to - a.window) : 0;
  return Range{start / kTile, (end + kTile - 1) / kTile, a.window > 0 ? max(0, end - a.window) : 0, whole_to};
}
// Steps of a piece: lengths are known here alone, and as many pieces as fill the chip should be about equal, whether one
// long sequence has them all or each sequence has its own.
__device__ __forceinline__ int keys_of(const AttendArgs& a, int b) {
  const long long held = (long long)a.table_width * a.block_size, seen = (long long)a.window + a.max_query_len;
  return max(0, (int)min((long long)a.seq_lens[b], a.window > 0 ? min(held, seen) : held));
}
template <int NC>
__device__ __forceinline__ int tiles_of(const AttendArgs& a, int b) {
  int queries = 1;
  if (a.query_start) {
    int row = a.query_start[b];
    queries = a.query_start[b + 1] - row;
    if (row < 0 || row > a.tokens) row = a.tokens;
    queries = min(max(0, min(queries, a.tokens - row)), a.max_query_len);
  }
  return (queries * a.group + 16 * NC - 1) / (16 * NC);
}
template <int NC>
__device__ __forceinline__ int steps_of_a_piece(const AttendArgs& a) {
  float all = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x & 63; i < a.seqs; i += 64) all += (float)keys_of(a, i) * (float)tiles_of<NC>(a, i);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) all += __shfl_xor(all, m);
  return __builtin_amdgcn_readfirstlane(max(a.least, (int)__builtin_ceilf(all * a.per_piece)));
}
// How many pieces a range of steps comes in (5/8: equal sequences, whose share is their number less a half, come in just
// that number).
__device__ __forceinline__ int pieces_of(const AttendArgs& a, int range, int steps) {
  return max(1, min(a.splits, (range + 5 * steps / 8) / steps));
}
// Which column tile and piece of which sequence is the unit'th of all; b = seqs behind the last.  The workgroups that
// have no work are so the last: between others they would keep CUs from these, since workgroups go to the CUs in turn
// (512 queries of 8 x 4 heads over 8192 keys 97 us, 186 with one for nothing beside each).
template <int NC>
__device__ __forceinline__ void find_piece(const AttendArgs& a, int unit, int steps, int& b, int& tile, int& split) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int first = 0; first < a.seqs; first += 64) {
    int pieces = 0, own = 0;
    if (first + lane < a.seqs) {  // (a window may begin and end inside a step: two more)
      pieces = a.splits == 1 ? 1 : pieces_of(a, keys_of(a, first + lane) / kTile + 2, steps);
      own = pieces * tiles_of<NC>(a, first + lane);
    }
    int upto = own;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int x = __shfl_up(upto, m);
      upto += lane >= m ? x : 0;
    }
    const uint64_t beyond = __ballot(before + upto > unit);
    if (beyond) {
      const int at = __builtin_ctzll(beyond);
      b = __builtin_amdgcn_readfirstlane(first + at);
      const int left = before + __builtin_amdgcn_readlane(upto, at) - 1 - unit;  // (tiles that see most come first)
      pieces = __builtin_amdgcn_readlane(pieces, at);
      tile = left / pieces;
      split = left - tile * pieces;
      return;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  b = a.seqs;
  tile = split = 0;
}

// The rows of a sequence past max_query_len were promised not to exist: they say so.
template <typename T, int D>
__device__ void refuse_rows(const AttendArgs& a, const Sequence& s, int kv) {
  const int per_row = a.group * D;
  for (int qi = a.max_query_len; qi < s.queries; ++qi) {
    T* dst = static_cast<T*>(a.out) + ((long long)(s.row + qi) * a.heads + kv * a.group) * D;
    for (int i = threadIdx.x; i < per_row; i += blockDim.x) dst[i] = (T)__builtin_nanf("");
  }
}

// Few queries a sequence: the waves of a workgroup share the keys of one column tile (or of one of `splits` pieces
// of them), joined through LDS; pieces are joined by a second kernel.  The reading of the cache bounds it: one token of
// 64 sequences of up to 4096 keys, 32 kv heads of 128, takes 114 us (5.1 TB/s; a kernel that only reads reaches 5.7), of 8
// sequences of up to 65536, 8 kv heads, 68 us (6.0) and 6 of the join.
template <typename T, int D, int NC, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, NC == 1 || D == 64 ? 3 : 2) attend_split_kernel(AttendArgs a) {
  constexpr int kCols = 16 * NC;
  __shared__ float part[WAVES][kCols][D + 4];
  __shared__ float maxima[WAVES][kCols], sums[WAVES][kCols];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = blockIdx.x / a.kv_heads, kv = blockIdx.x - unit * a.kv_heads;
  Wave<T, D, NC, NC == 1> w(a);  // (16 columns are all there are, or all that is small)
  int b = unit, tile = gridDim.y - 1 - blockIdx.y, split = 0, steps = 1;  // (tiles that see most come first)
  // Without a window the keys begin where they do whatever the length, which is under way meanwhile: one round trip to
  // memory less before the first keys.
  // Workgroups go to the CUs in turn: sequences in the same order in each row of tiles would give the long ones to the same
  // CUs again and again (2 x 1024 queries of 8 x 4 heads over 2500 and 8192 keys 269 us, 344 so).
  if (!a.search && gridDim.y > 2) b = (int)((unsigned)(unit + ((tile * 40503u) >> 5)) % (unsigned)a.seqs);
  const bool ahead = a.window == 0 && !a.search;  // (few tiles are without queries then)
  if (__builtin_expect(a.search, 0)) {
    if (a.splits > 1) steps = steps_of_a_piece<NC>(a);
    find_piece<NC>(a, unit, steps, b, tile, split);
    if (b == a.seqs) return;
  }
  if (ahead) w.first_loads(b, kv, wave, &part[wave][0][0]);
  const Sequence s = sequence(a, b);
  const int queries = min(s.queries, a.max_query_len), cols = queries * a.group;
  if (tile == 0 && split == 0 && queries < s.queries) refuse_rows<T, D>(a, s, kv);
  const int col0 = tile * kCols;
  if (col0 >= cols) return;
  const Range r = range(a, s, col0, min(cols - 1, col0 + kCols - 1));
  const int all = r.last_tile - r.first_tile, pieces = a.splits == 1 ? 1 : pieces_of(a, all, steps);
  if (split >= pieces) return;
  const int t0 = r.first_tile + all * split / pieces + wave, t1 = r.first_tile + all * (split + 1) / pieces;
  if (!ahead) w.first_loads(b, kv, t0, &part[wave][0][0]);
  w.begin(s, kv, col0, cols);
  w.template run<false>(t0, t1, WAVES, s.length, r.whole_from, r.whole_to);

  w.set_aside();
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const float total = over_groups_sum(w.kept_sum[n]);
    if (w.g == 0) {
      maxima[wave][16 * n + w.c] = -w.shift[n];
      sums[wave][16 * n + w.c] = total;
    }
  }
  __syncthreads();
  constexpr int kEach = D * kCols / (64 * WAVES);  // elements of a column that a thread joins
  constexpr int kPer = D / kEach;
  const int col = threadIdx.x / kPer, d0 = (threadIdx.x % kPer) * kEach;
  if (col0 + col >= cols) return;
  float top = maxima[0][col];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) top = fmaxf(top, maxima[i][col]);
  float total = 0.f, x[kEach] = {};
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const float f = exp2_(maxima[i][col] - top);
    total = __builtin_fmaf(sums[i][col], f, total);
#pragma unroll
    for (int d = 0; d < kEach; ++d) x[d] = __builtin_fmaf(part[i][col][d0 + d], f, x[d]);
  }
  const int qi = (col0 + col) / a.group, head = kv * a.group + (col0 + col) - qi * a.group;
  const long long at = (long long)(s.row + qi) * a.heads + head;
  if (pieces == 1) {
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

// Joins the pieces of a query head: one wave each, a lane a piece for the factors, then 16 bytes a lane of several
// pieces at once.
template <typename T, int D, int NC>
__global__ void __launch_bounds__(256) attend_join_kernel(AttendArgs a) {
  const int at = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (at >= a.tokens * a.heads) return;
  const int row = at / a.heads, kv = (at - row * a.heads) / a.group;
  int b = row;
  if (a.query_start) {  // the last sequence that begins at or before this row
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (scalar(a.query_start)[mid] <= row)
        lo = mid;
      else
        hi = mid;
    }
    b = lo;
  }
  const Sequence s = sequence(a, b);
  const int qi = row - s.row, queries = min(s.queries, a.max_query_len);
  if (qi < 0 || qi >= queries) return;  // a row of no sequence, or one past max_query_len: neither is written here
  const int cols = queries * a.group, col = qi * a.group + (at - row * a.heads) - kv * a.group;
  const int col0 = col / (16 * NC) * (16 * NC);
  const Range r = range(a, s, col0, min(cols - 1, col0 + 16 * NC - 1));
  const int pieces = pieces_of(a, r.last_tile - r.first_tile, steps_of_a_piece<NC>(a));
  if (pieces == 1) return;  // written by the first kernel
  constexpr int kLanes = D / 4, kAtOnce = 64 / kLanes;
  const int lane = threadIdx.x & 63, part = lane / kLanes, d = 4 * (lane % kLanes);
  const float* ml = a.part_ml + (long long)at * a.splits * 2;
  float most = kNone, total = 0.f;
  if (lane < pieces) most = ml[2 * lane], total = ml[2 * lane + 1];
  float top = most;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
  const float f = lane < pieces ? exp2_(most - top) : 0.f;
  total *= f;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) total += __shfl_xor(total, m);
  const float* src = a.part_o + (long long)at * a.splits * D + d;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < pieces; i += kAtOnce) {
    const int piece = i + part;
    const float fp = __shfl(f, piece & 63);
    if (piece < pieces) x += *reinterpret_cast<const f32x4*>(src + (long long)piece * D) * fp;
  }
#pragma unroll
  for (int m = kLanes; m < 64; m <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], m);
  if (part) return;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  vec4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (T)(total == 0.f ? 0.f : x[i] / total);
  *reinterpret_cast<vec4*>(static_cast<T*>(a.out) + (long long)at * D + d) = y;
}

// The sequence of the rank'th greatest length, of up to 64 (more fill the chip however they come).
__device__ __forceinline__ int by_length(const AttendArgs& a, int rank) {
  if (a.seqs > 64) return rank;
  const int lane = threadIdx.x & 63;
  const int own = lane < a.seqs ? a.seq_lens[lane] : -0x7fffffff;
  int ahead = 0;
  for (int i = 0; i < a.seqs; ++i) {
    const int other = __builtin_amdgcn_readlane(own, i);
    ahead += other > own || (other == own && i < lane);
  }
  return __builtin_ctzll(__ballot(ahead == rank && lane < a.seqs));
}

// Many queries a sequence: each wave has columns of its own and runs over all the keys that they see; the four waves of
// a workgroup hold neighbouring columns, so that they read the same keys at about the same time.  Vector instructions
// bound it (261 and 16 exponentials for 32 matrix instructions in bf16, 293 and 16 for 34 in fp16): 2 x 2048 queries of 64
// heads of 128 over 2500 and 8192 keys take 712 us (770 in fp16), 0.77 PFLOP/s.  Converting each code once a workgroup,
// through LDS, takes a quarter of them away and costs more in waits than that (740 us with two barriers a step).
template <typename T, int D, int NC>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) attend_prompt_kernel(AttendArgs a) {
  constexpr int kCols = 16 * NC;
  __shared__ float part[4][kCols][D + 4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv = blockIdx.x, b = by_length(a, blockIdx.z);
  const Sequence s = sequence(a, b);
  const int queries = min(s.queries, a.max_query_len), cols = queries * a.group;
  if (blockIdx.y == 0 && queries < s.queries) refuse_rows<T, D>(a, s, kv);
  const int group_cols = 4 * kCols, groups = (cols + group_cols - 1) / group_cols;
  if ((int)blockIdx.y >= groups) return;
  // the columns that see most come first: what is left at the end is short
  const int col0 = (groups - 1 - (int)blockIdx.y) * group_cols + wave * kCols;
  if (col0 >= cols) return;
  const Range r = range(a, s, col0, min(cols - 1, col0 + kCols - 1));
  Wave<T, D, NC, false> w(a);
  w.first_loads(b, kv, r.first_tile, &part[wave][0][0]);
  w.begin(s, kv, col0, cols);
  w.template run<true>(r.first_tile, r.last_tile, 1, s.length, r.whole_from, r.whole_to);
  if (w.keeps) w.set_aside();
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const float total = over_groups_sum(w.keeps ? w.kept_sum[n] : w.sum[n]);
    const int col = col0 + 16 * n + w.c;
    const int qi = col / a.group, head = kv * a.group + col - qi * a.group;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    w.results(n, [&](int d, float* x) {
      if (col >= cols) return;
      if (w.keeps) {  // (the registers were set aside and hold nothing)
        const f32x4* at = reinterpret_cast<const f32x4*>(&part[wave][16 * n + w.c][d]);
#pragma unroll
        for (int m = 0; m < D / 16; ++m) x[m] = at[m / 4][m % 4];
      }
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
  int nc, tiles, waves, search, splits, least;
  long long units;
  float per_piece;
};
Plan plan(int tokens, int seqs, int heads, int kv_heads, int max_query_len, int max_seq_len, int window, int head_size) {
  const long long group = heads / kv_heads, cols = max_query_len * group;
  Plan p;
  p.waves = 4;
  p.search = 0;
  p.splits = 1;
  p.least = 1;
  p.per_piece = 1.f;
  p.units = seqs;
  // Column tiles of nc x 16, and those of them that hold queries: of all rows together (a batch may mix one prompt with
  // many single tokens), a tile a sequence more where they do not fill their last.
  long long most_tiles, full, tiles, groups;
  const auto tile = [&](int nc) {
    p.nc = nc;
    p.tiles = (int)((cols + 16 * nc - 1) / (16 * nc));
    most_tiles = (long long)seqs * p.tiles;
    full = max_query_len == 1 ? most_tiles : (tokens * group + 16 * nc - 1) / (16 * nc);
    tiles = full + seqs < most_tiles ? full + seqs : most_tiles;
    groups = tiles * kv_heads;
  };
  tile(cols > 16 ? 2 : 1);
  // A wave for each column tile where these alone fill the chip, two waves a SIMD, and the rows are spread about evenly:
  // 2 x 8 kv heads x 1024 queries of 8 heads take 70 us so and 98 with waves that share the keys, 64 x 8 x 32 queries of
  // 4 heads over 1024 keys 60 and 71.  Below that some SIMDs idle while others have all the keys to run over: one
  // sequence's 512 queries of 8 x 4 heads over 8192 keys 268 and 102, one query of 128 heads over 65536 keys 2070 and 27;
  // 2048 queries beside 63 single ones, each over 4096 keys, 995 and 222.  Long sequences want a second such round
  // (2048 queries of 8 x 4 heads over 65536 keys, one round: 2970 and 2710; twice 2048 over 8192, two: 633 and 630).
  // (A grid takes 65535 in the direction that its sequences, and its groups of four tiles, have to themselves.)
  p.prompt = cols > 64 && full * kv_heads >= (max_seq_len > 2048 ? 4096 : 2048) && 2 * full >= most_tiles && seqs <= 65535;
  if (p.prompt) return p;
  long long keys = max_seq_len;
  if (window > 0 && (long long)window + max_query_len < keys) keys = window + max_query_len;
  // Where a workgroup a CU is all there is eight waves share the keys, up to 2048 of them without a second kernel (16 x 4
  // kv heads x 1029 keys of 64 take 11.8 us so, 14.6 with four waves and two pieces), more in pieces of 512 (8 kv heads x
  // 4096 keys of 128 13.0 us; of 256 12.7, of 1024 14.7, of 2048 18.7; of 32 x 4096 14.7, 14.7, 15.5 and 19.3).
  // Otherwise as many pieces as fill the chip once: four workgroups of four waves a CU, three for heads of 128, two of 32
  // columns, which is what their registers allow (2 x 32 x 56000 keys of 64 60 us; in three or five a CU 63).
  const long long rounds = (keys + 2047) / 2048;
  if (p.nc == 2 && groups * rounds <= 256) {
    // ... and tiles of 16 columns spread the work wider where they fit too: 16 x 4 kv heads x 5 queries of 7 heads over 1024
    // keys of 64 9.0 us against 11.9, one query of 128 heads over 2000 keys of 128 14.4 against 19.4; of half as many
    // again no more (8 x 8 x 64 columns over 4096 keys 39.8 and 38.1).
    tile(1);
    if (groups * rounds > 256) tile(2);
  }
  if (groups * rounds <= 256) p.waves = 8;
  const long long fill = p.nc == 2 ? 512 : head_size == 64 ? 1024 : 768;
  // More short sequences than fill the chip once take fewer waves each, so that it holds more of them: 1024 x 250 keys of
  // 128 10.4 us with two waves, 13.7 with four, 11.7 with one; 2048 x 129 16.9, 21.5 and 12.6, x 500 30.2, 31.3 and 25.0;
  // 4 x 500 queries of 8 x 4 heads 29.9, 41.4 and 27.4.
  if (keys <= (p.nc == 2 ? 1024 : 512) && groups > fill) p.waves = groups > 2 * fill ? 1 : 2;
  // Rows that are spread unevenly would leave workgroups without work, which are looked past: 512 queries beside 63 single
  // ones, each over 4096 keys, 115 us and 252.
  p.search = tiles < most_tiles;
  p.units = p.search ? tiles : seqs;
  if (keys <= (p.waves == 8 ? 2048 : p.waves == 4 ? 512 : 1024)) return p;
  const long long least = 512, most = (keys + least - 1) / least;
  long long cut = (p.waves == 8 ? 256 : fill) / groups;
  cut = cut < 1 ? 1 : cut;
  // A long sequence among short ones comes in more, at what looking for the pieces and a second kernel cost the others:
  // 63 x 500 keys of 8 kv heads beside one of 65536 take 38 us so and 395 with a workgroup each, 64 lengths spread over
  // their logarithm up to 32768 67 and 194, 64 x 4096 49 and 45.  Where sequences fill the chip several times over there
  // is less to even out than that costs, and so where the longest are short: 256 lengths of up to 16384 152 and 191,
  // 256 x 2048 111 and 90, 127 x 800 35 and 25.  (What is not taken up of a workspace costs nothing; it stays below 2^18
  // pieces of a query head.)
  const long long room = (1LL << 18) / ((long long)tokens * heads);
  long long splits = cut == 1 && (groups > 1024 || keys <= 2048 || seqs == 1) ? 1 : most < room ? most : room;
  p.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
  p.least = (int)(least / kTile);
  if (p.splits == 1) return p;
  // (half a piece a tile for the rounding of their numbers: one workgroup too many is a round too many)
  p.per_piece = 1.f / ((float)kTile * (float)tiles * (cut == 1 ? 1.f : (float)cut - 0.5f));
  // At most one piece a tile more than its share, and 2 / 16 for the two steps that are added to it.
  p.search = 1;
  p.units = tiles * (cut + 1) + (tiles + 3) / 4;
  return p;
}

template <typename T, int D>
int launch(const AttendArgs& a, const Plan& p, hipStream_t s) {
  if (p.prompt) {
    // the longest sequence first, and of each the columns that see most: the short ones fill the end.  In one order for
    // all, 2 x 2048 queries that see up to 2500 and 8192 keys leave 40 % of the CUs' time unused.  A kv head's workgroups
    // follow each other at a distance of kv_heads, which puts them on the same XCD where that is 8.
    const dim3 grid((unsigned)a.kv_heads, (unsigned)((p.tiles + 3) / 4), (unsigned)a.seqs);
    hipLaunchKernelGGL((attend_prompt_kernel<T, D, 2>), grid, dim3(256), 0, s, a);
    return serving_after_launch();
  }
  const dim3 grid((unsigned)(p.units * a.kv_heads), p.search ? 1u : (unsigned)p.tiles);
  if (p.nc == 1 && p.waves == 1)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 1, 1>), grid, dim3(64), 0, s, a);
  else if (p.nc == 1 && p.waves == 2)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 1, 2>), grid, dim3(128), 0, s, a);
  else if (p.nc == 1 && p.waves == 4)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 1, 4>), grid, dim3(256), 0, s, a);
  else if (p.nc == 1)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 1, 8>), grid, dim3(512), 0, s, a);
  else if (p.waves == 1)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 2, 1>), grid, dim3(64), 0, s, a);
  else if (p.waves == 2)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 2, 2>), grid, dim3(128), 0, s, a);
  else if (p.waves == 4)
    hipLaunchKernelGGL((attend_split_kernel<T, D, 2, 4>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attend_split_kernel<T, D, 2, 8>), grid, dim3(512), 0, s, a);
  int rc = serving_after_launch();
  if (rc != SERVING_OK || p.splits == 1) return rc;
  const dim3 join((unsigned)(((long long)a.tokens * a.heads + 3) / 4));
  if (p.nc == 1)
    hipLaunchKernelGGL((attend_join_kernel<T, D, 1>), join, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attend_join_kernel<T, D, 2>), join, dim3(256), 0, s, a);
  return serving_after_launch();
}

size_t workspace_of(const Plan& p, int tokens, int heads, int head_size) {
  return p.splits == 1 ? 0 : (size_t)tokens * heads * p.splits * (head_size + 2) * sizeof(float);
}

bool sizes_ok(int tokens, int seqs, int heads, int kv_heads, int max_query_len, int max_seq_len, int window) {
  return tokens > 0 && seqs > 0 && heads > 0 && heads <= 65535 && kv_heads > 0 && kv_heads <= heads && heads % kv_heads == 0 &&
         max_query_len > 0 && max_seq_len > 0 && max_seq_len <= (1 << 27) && window >= 0;
}

// What a plan can count in: rows and heads, sequences and kv heads.
bool countable(int tokens, int seqs, int heads, int kv_heads) {
  return (long long)seqs * kv_heads <= 0x7fffffLL && (long long)tokens * heads <= 0x7fffffffLL;
}

}  // namespace

extern "C" size_t serving_attend_kv4_workspace_bytes(int tokens, int seqs, int heads, int kv_heads, int head_size,
                                                     int max_query_len, int max_seq_len, int window) {
  if (!sizes_ok(tokens, seqs, heads, kv_heads, max_query_len, max_seq_len, window) || !head_size_ok(head_size) ||
      !countable(tokens, seqs, heads, kv_heads))
    return 0;
  max_query_len = max_query_len < tokens ? max_query_len : tokens;  // (no sequence has more rows than there are)
  const Plan p = plan(tokens, seqs, heads, kv_heads, max_query_len, max_seq_len, window, head_size);
  return workspace_of(p, tokens, heads, head_size);
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
  if (!countable(tokens, seqs, heads, kv_heads)) return SERVING_E_TOO_LARGE;
  max_query_len = max_query_len < tokens ? max_query_len : tokens;
  const Plan p = plan(tokens, seqs, heads, kv_heads, max_query_len, max_seq_len, window, head_size);
  if ((!p.search && p.tiles > (p.prompt ? 4 : 1) * 65535LL) ||
      (!p.prompt && p.units * kv_heads * p.waves * 64 > 0xffffffffLL))
    return SERVING_E_TOO_LARGE;
  const size_t need = workspace_of(p, tokens, heads, head_size);
  if (need && (!workspace || workspace_bytes < need)) return SERVING_E_WORKSPACE;
  if (need && !aligned16(workspace)) return SERVING_E_ALIGN;
  const int sixteens = block_size / 16;
  AttendArgs a{query, q_token, q_head, static_cast<const uint8_t*>(cache), tables, table_stride, seq_lens, query_start, out,
               static_cast<float*>(workspace), nullptr, table_width, tokens, seqs, heads, kv_heads, heads / kv_heads,
               (int)num_blocks, block_size,
               sixteens == 1 ? 0u : (uint32_t)(((1ULL << 32) + sixteens - 1) / sixteens),
               scale * 1.44269504088896340736f, window, max_query_len, p.search, p.splits, p.least, p.per_piece};
  if (need) a.part_ml = a.part_o + (size_t)tokens * heads * p.splits * head_size;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_size == 64) return bf16_in ? launch<bf16, 64>(a, p, s) : launch<f16, 64>(a, p, s);
  return bf16_in ? launch<bf16, 128>(a, p, s) : launch<f16, 128>(a, p, s);
}
