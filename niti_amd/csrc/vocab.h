// Losses over a large vocabulary (vocab.hip, vocab_rows.hip): what their launchers share.
//
// a [N][F] and w [V][F] are int8 with exponents ea, ew; s = a . w is the exact int32 product, z = s 2^(ea + ew) / T a logit.
// All exponentials are powers of two: with k = 2^(ea + ew) log2(e) / T a row's softmax is
//   p_v = 2^((s_v - m) k - L),  m = max_v s_v (an integer: the differences are exact),  L = log2 sum_v 2^((s_v - m) k).
// A row with targets q_j at the classes i_j (one of weight 1 for an entropy, the teacher's for a distillation) has the logit gradient
//   g_v = T (p_v sum_j q_j - sum_{j: i_j = v} q_j),
// the activations' d_a = weight_n (g . w) 2^ew and the weights' d_w = ((weight g)^T . a) 2^ea.
#pragma once
#include "common.h"

namespace niti {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// p and g lie in [-1, 1]; as 16-bit floats they are kept times 2^15: eleven significant bits down to 2^-29, where bfloat16 has eight
constexpr int kGradExponent = 15;
// rows of the weight gradient's left operand: activation times row weight over the power of two above the largest row weight, times 2^8
constexpr int kRowExponent = 8;
constexpr int kVocabTopMost = 1024;      // places of a teacher's list (one row's are kept in LDS)

// What a forward pass leaves of a row: m, L (float), the sum of the targets' weights (float: 1; 0, nothing to learn from; NaN,
// undefined), a word of nothing, then for each of its `top` places g / T (float) and the class, -1 where there is none or an earlier place
// has named it.  Rows start on 16 bytes.
inline __host__ __device__ long long vocab_state_words(int top) { return 4 + (2LL * top + 3) / 4 * 4; }

// One operand of a product tile: rows of `pitch` bytes, 4-byte aligned.
//   reduction index fast: `rows` rows of `row_bytes` readable bytes; where these are no multiple of 16, sixteen bytes at a row's end hold
//   the beginning of what follows, and the other operand is zero there
//   reduction index slow: `rows` steps of the reduction, tile columns along the row, whose readable length is row_bytes
struct VocabOperand {
  const void* p;
  long long pitch;
  int rows;
  int row_bytes;
};

struct VocabLogits {         // s[v][n] = w[v] . a[n]
  VocabOperand w, a;         // reduction fast in both
  int classes, rows, features;
  const int32_t* exp_a;
  const int32_t* exp_w;
  float inv_t;               // 1 / T
};

struct VocabStats {          // (max, sum of 2^((s - max) k)) of each row over each tile's classes
  int2* part;                // [rows][tiles]
  int tiles;
};

// What a row learns from, and the logits there (sums of products as they are): made by workgroups of the statistics' launch
struct VocabTargets {
  const void* index;         // [rows][top] int32 or int64
  int index_bytes;
  int distill;               // 0: entropy
  long long ignored;         // entropy: this class is none; distillation: every negative one
  int top;
  int32_t* state;            // receives a place's logit where its gradient will be; what an unused place receives means nothing
};
// class of a place: -1 none, -2 outside of the classes
__device__ inline int vocab_target(const VocabTargets& t, long long at, int classes) {
  const long long c = t.index_bytes == 8 ? static_cast<const int64_t*>(t.index)[at] : static_cast<const int32_t*>(t.index)[at];
  if (t.distill ? c < 0 : c == t.ignored) return -1;
  return c >= 0 && c < classes ? static_cast<int>(c) : -2;
}

// A grid's work-items are counted in 32 bits.
inline int check_grid(long long workgroups, int threads, const char* what) {
  if (workgroups > 0xffffffffLL / threads) return fail(NITI_ERR_UNSUPPORTED, "%s: %lld workgroups of %d", what, workgroups, threads);
  return NITI_OK;
}

// Sums and maxima over the wavefront by data-parallel moves (a scan inside each row of sixteen lanes, the row totals carried on), in every
// lane: six moves of a few clocks where a shuffle through LDS is some hundred.
template <int CTRL, int MASK>
__device__ inline int dpp_take(int neutral, int v) { return __builtin_amdgcn_update_dpp(neutral, v, CTRL, MASK, 0xf, false); }
template <class F>
__device__ inline int wave_fold(int neutral, int v, F f) {
  v = f(v, dpp_take<0x111, 0xf>(neutral, v));
  v = f(v, dpp_take<0x112, 0xf>(neutral, v));
  v = f(v, dpp_take<0x114, 0xf>(neutral, v));
  v = f(v, dpp_take<0x118, 0xf>(neutral, v));
  v = f(v, dpp_take<0x142, 0xa>(neutral, v));
  v = f(v, dpp_take<0x143, 0xc>(neutral, v));
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ inline int wave_add(int v) {
  return wave_fold(0, v, [](int a, int b) { return a + b; });
}
__device__ inline int wave_most(int v) {
  return wave_fold(-2147483647 - 1, v, [](int a, int b) { return max(a, b); });
}
__device__ inline float wave_add(float v) {
  return __int_as_float(wave_fold(0, __float_as_int(v), [](int a, int b) { return __float_as_int(__int_as_float(a) + __int_as_float(b)); }));
}
// in 64 bits: the two halves move together
template <int CTRL, int MASK>
__device__ inline double dpp_take(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const int lo = dpp_take<CTRL, MASK>(0, static_cast<int>(b)), hi = dpp_take<CTRL, MASK>(0, static_cast<int>(b >> 32));
  return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo)));
}
__device__ inline double wave_add(double v) {
  v += dpp_take<0x111, 0xf>(v);
  v += dpp_take<0x112, 0xf>(v);
  v += dpp_take<0x114, 0xf>(v);
  v += dpp_take<0x118, 0xf>(v);
  v += dpp_take<0x142, 0xa>(v);
  v += dpp_take<0x143, 0xc>(v);
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const int lo = __builtin_amdgcn_readlane(static_cast<int>(b), 63), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), 63);
  return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo)));
}
__device__ inline float wave_most(float v) {
  return __int_as_float(wave_fold(__float_as_int(-INFINITY), __float_as_int(v), [](int a, int b) { return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b))); }));
}

// int8 rows to 16-bit floats, each times weight / 2^*exponent 2^kRowExponent where there are weights; *exponent receives the smallest power of
// two above every weight
struct VocabWiden {
  const int8_t* src;         // rows of src_bytes readable bytes, 4-byte aligned; what is made of bytes behind `values` means nothing
  long long src_pitch;
  int src_bytes;
  _Float16* dst;
  long long pitch;
  int rows, values;
  const float* weight;
  int32_t* exponent;
  int blocks;                // 0: nothing to do
};

struct VocabGrad {           // sum_j q_j p, times 2^kGradExponent, of the classes of a piece
  const int32_t* state;      // [rows][state_words]
  long long state_words;
  int top;                   // targets written into the piece here; 0: vocab_targets_kernel does it
  long long first;           // class that the piece starts at
  _Float16* g;               // [rows][pitch], zero between the piece's last class and the next multiple of eight
  long long pitch;
  VocabWiden widen_a, widen_w;   // done by workgroups of their own
};

struct VocabSums {           // out[j][i] = sum_k x[i][k] y[j][k] in float
  VocabOperand x, y;
  int ni, nj, nk;
  int slices, steps;         // reduction cut in `slices` parts of `steps` stages of 64
  float* part;               // [slices][nj][part_pitch]; null: written to out at once
  long long part_pitch;
  int accumulate;            // add to what part holds
  uint16_t* out;             // bfloat16 [nj][ni]
  float* out32;              // the same in float32 in its place, where it is not null (then part is not, either)
  // scale of the result: T 2^(exponent) weight
  float t;
  const int32_t* exponent;
  int bias;
  const int32_t* exponent2;  // may be null
  const float* weight;       // per j; null: 1.  weight_n == 1: the same for all
  int weight_n;
};

// The tiles of a launch (vocab.hip): 256 x 256; 128 x 128 two to a unit; 64 x 64; short, the sums of few rows (64 x 64 for the activations, one
// buffer of 128 x 128 for the weights); 32 rows; 128 x 128 in one buffer, four to a unit; 64 x 64 and, of 32 rows, 64 x 32 whose wavefronts take
// stages of their own
// (niti_vocab_plan gives their numbers out)
enum VocabTile { kVocabLarge, kVocabMiddle, kVocabSmall, kVocabShort, kVocabFew, kVocabQuad, kVocabSmallApart, kVocabFewApart };
VocabTile vocab_logits_tile(int rows, int features, int classes);
int vocab_stats_tiles(VocabTile t, int classes);    // pairs that launch_vocab_stats leaves of a row
bool vocab_sums_wants_wide_weights(VocabTile t);
bool vocab_grad_writes_targets(VocabTile t, int top);
int launch_vocab_stats(VocabTile t, const VocabLogits& l, const VocabStats& s, const VocabTargets& targets, hipStream_t stream);
int launch_vocab_grad(VocabTile t, const VocabLogits& l, const VocabGrad& g, hipStream_t stream);
// Both gradients' sums of a piece: a = the activations' (x: weights, int8 or a 16-bit copy, reduction slow; y: the piece's gradient, reduction fast), w = the
// weights' (x: 16-bit activations, y: the piece's gradient, reduction slow in both)
VocabTile vocab_sums_plan(int rows, int features, int classes, int* slices_a, int* steps_a, int* slices_w, int* steps_w);
int launch_vocab_sums(VocabTile t, const VocabSums& a, const VocabSums& w, hipStream_t stream);
int launch_vocab_join(const VocabSums* a, const VocabSums* w, hipStream_t stream);   // either may be null; those that write float32 go through here

}  // namespace niti
