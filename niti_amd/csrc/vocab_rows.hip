// Losses over a large vocabulary (vocab.h): what is done per row, the operands' layouts, and the entry points.
//
//   forward:  statistics of the logits per row and tile of classes and the logits of the targets (vocab.hip), then a wavefront per row
//             joins them and leaves loss, logarithm of the denominator and what the backward pass wants to know
//   backward: a piece of the classes after the other: the piece's softmax as 16-bit floats (vocab.hip), the targets' places
//             overwritten with their gradient (made in 32 bits: a difference p - q keeps what its rounding leaves, p - 1 its digits), both
//             products in one launch, their slices added in another
#include <math.h>

#include "vocab.h"

namespace niti {
namespace {

constexpr int kMaxFeatures = 65536;      // |s| <= 2^30: differences of two logits are int32
constexpr int kMaxRows = (1 << 26) - 1;  // a wavefront each in one launch
constexpr long long kPieceMost = 1LL << 20;
// A piece of the classes: as many as leave the gradient at 128 MiB, half of the last-level cache, and the weights' 16-bit copy at 256 MiB, but 4096 at
// least.  Rows are not cut: from 16384 on the gradient is 8 KiB of each, whatever the cache holds, and from 32768 features on the weights' copy 8 KiB of each
// feature.  Every piece adds to all of d_act's float32 sums, so fewer classes cost more than they save: 131072 rows over 32000 classes 8.3 ms at
// 256 features and 11.7 at 512 with 4096 classes, 14.8 and 17.1 with 512 and 1024.
constexpr long long kPieceGrad = 64LL << 20;    // values
constexpr long long kPieceWide = 128LL << 20;   // values
constexpr long long kPieceLeast = 4096;         // classes

long long round_up(long long v, long long to) { return (v + to - 1) / to * to; }

// ---- layouts -------------------------------------------------------------------------------------------------------
// Rows of `n` bytes at any address and pitch -> rows of a multiple of 16, zero behind the last byte; up to two matrices in a launch.  Reads
// whole words that hold at least one byte of the row, and puts sixteen bytes together from five of them.  20011 rows of 997
// bytes 9.7 us, 4.1 TB/s there and back.
struct VocabPad {
  const int8_t* src;
  long long pitch;
  int8_t* dst;
  long long rows;
  int blocks;
};
__global__ __launch_bounds__(256) void vocab_pad_kernel(const VocabPad a, const VocabPad b, int n) {
  const bool first = static_cast<int>(blockIdx.x) < a.blocks;
  const VocabPad p = first ? a : b;
  const int pieces = (n + 15) / 16;
  const long long at = static_cast<long long>(blockIdx.x - (first ? 0 : a.blocks)) * 256 + threadIdx.x, all = p.rows * pieces;
  if (at >= all) return;
  const long long row = all < 0x7fffffffLL ? static_cast<unsigned>(at) / static_cast<unsigned>(pieces) : at / pieces;
  const int c = static_cast<int>(at - row * pieces) * 16;
  const uintptr_t from = reinterpret_cast<uintptr_t>(p.src + row * p.pitch + c);
  const uint32_t* const words = reinterpret_cast<const uint32_t*>(from & ~static_cast<uintptr_t>(3));
  const int skip = static_cast<int>(from & 3), bytes = min(16, n - c);
  uint32_t w[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = 4 * i < skip + bytes ? words[i] : 0u;
  v4i o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v = static_cast<uint32_t>(((static_cast<uint64_t>(w[i + 1]) << 32) | w[i]) >> (8 * skip));
    const int in = bytes - 4 * i;       // bytes of this word that are the row's
    if (in < 4) v &= in <= 0 ? 0u : (1u << (8 * in)) - 1u;
    o[i] = static_cast<int>(v);
  }
  *reinterpret_cast<v4i*>(p.dst + at * 16) = o;
}

// ---- rows ------------------------------------------------------------------------------------------------------------
struct VocabRows {
  const int2* part;           // [rows][tiles]
  int tiles;
  int rows, classes;
  const int32_t* exp_a;
  const int32_t* exp_w;
  float t;
  VocabTargets targets;
  const void* value;          // [rows][top] teacher's logits; null: entropy
  int value_type;
  float* loss;
  float* lse;
  int32_t* state;
};

__device__ inline float teacher_value(const VocabRows& a, long long i) {
  if (a.value_type == NITI_F32) return static_cast<const float*>(a.value)[i];
  if (a.value_type == NITI_BF16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(a.value)[i]) << 16);
  return static_cast<float>(static_cast<const _Float16*>(a.value)[i]);
}

// A wavefront and workgroup per row.  All loads depend on nothing and go out together: pairs of the tiles, exponents, targets, their logits
// and teacher's values; what the kernel takes is the way of these.  3.0 us for one row, 4.0 for 128, 20 for 8192 rows with 64
// places.  The tiles' sums, of 32 bits, are added in 64: a row that is all but sure of itself adds many small ones to one that is almost 1, and what they
// come to is its loss.  A logit's distance from the largest and the logarithm of the sum meet in 64 bits.
__global__ __launch_bounds__(64) void vocab_rows_kernel(const VocabRows a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;
  const int top = a.targets.top;
  float* const q = reinterpret_cast<float*>(smem);
  int* const cls = reinterpret_cast<int*>(q + top);

  constexpr int kHeld = 4;            // pairs in registers; a row of more tiles is read twice
  const int2* const part = a.part + row * a.tiles;
  int2 held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) held[u] = lane + 64 * u < a.tiles ? part[lane + 64 * u] : make_int2(-2147483647 - 1, 0);
  const int exponent = *a.exp_a + *a.exp_w;
  int32_t* const state = a.state + row * vocab_state_words(top);      // a place's gradient takes the place of its logit
  const int dot0 = lane < top ? state[4 + 2 * lane] : 0;

  // the targets and their weights
  bool bad = false;
  float vmax = -INFINITY;
  for (int j = lane; j < top; j += 64) {
    const long long at = row * top + j;
    const int c = vocab_target(a.targets, at, a.classes);
    const float given = a.value == nullptr ? 0.0f : teacher_value(a, at);
    if (c == -2) bad = true;
    cls[j] = c < 0 ? -1 : c;
    const float v = c < 0 ? -INFINITY : given;
    q[j] = v;
    vmax = fmaxf(vmax, v);
  }

  // the denominator
  const double k = fmin(ldexp(1.4426950408889634074 / static_cast<double>(a.t), exponent), 3.402823466e38);
  const float kf = static_cast<float>(k);
  int m = -2147483647 - 1;
#pragma unroll
  for (int u = 0; u < kHeld; ++u) m = max(m, held[u].x);
  for (int i = lane + 64 * kHeld; i < a.tiles; i += 64) m = max(m, part[i].x);
  m = wave_most(m);
  double sum = 0.0;
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (held[u].x != -2147483647 - 1) sum += __int_as_float(held[u].y) * exp2f(static_cast<float>(held[u].x - m) * kf);
  for (int i = lane + 64 * kHeld; i < a.tiles; i += 64) {
    const int2 v = part[i];
    sum += __int_as_float(v.y) * exp2f(static_cast<float>(v.x - m) * kf);
  }
  sum = wave_add(sum);
  int e2;
  double mantissa = frexp(sum, &e2);
  if (mantissa < 0.70710678) {
    mantissa *= 2.0;
    e2 -= 1;
  }
  // the float part is at most 1/2, and what the mantissa has beyond float counts by the logarithm's slope at 1: a row that is sure of itself keeps its digits
  const float rounded = static_cast<float>(mantissa);
  const double l2 = 1.4426950408889634074 * (mantissa - rounded) + log2f(rounded) + e2;

  vmax = wave_most(vmax);
  bad = __any(bad);
  float norm = 0.0f;
  for (int j = lane; j < top; j += 64) {
    const float v = q[j];
    // divided by T behind the difference: a type's lowest value over a T below 1 is no float32 number any more, its difference from another is
    const float e = v == -INFINITY ? 0.0f : expf((v - vmax) / a.t);
    q[j] = e;
    norm += e;
  }
  norm = wave_add(norm);
  const float coef = bad ? __builtin_nanf("") : (norm > 0.0f ? 1.0f : (norm == 0.0f ? 0.0f : __builtin_nanf("")));
  __syncthreads();

  constexpr double kLn2 = 0.69314718055994530942;
  float loss = 0.0f;
  for (int j = lane; j < top; j += 64) {
    const int c = cls[j];
    float g = 0.0f;
    bool first = c >= 0;
    if (c >= 0) {
      const float mine = q[j] / norm;
      const double behind = (static_cast<double>(j < 64 ? dot0 : state[4 + 2 * j]) - m) * k - l2;       // log2 of the softmax here
      if (mine > 0.0f) loss += mine * (logf(mine) - static_cast<float>(kLn2 * behind));
      else if (!(mine == 0.0f)) loss = mine;
      float all = 0.0f;                  // the weights of every place that names this class
      for (int i = 0; i < top; ++i)
        if (cls[i] == c) {
          all += q[i];
          if (i < j) first = false;      // one place speaks for all
        }
      // p near 1 by its distance from 1: what p - 1 is of a row that is all but sure of itself has its own digits, not those that 1 leaves
      if (norm > 0.0f) g = behind > -1.0 ? expm1f(static_cast<float>(kLn2 * behind)) + (norm - all) / norm : exp2f(static_cast<float>(behind)) - all / norm;
      if (coef != coef) g = coef;
    }
    *reinterpret_cast<int2*>(state + 4 + 2 * j) = make_int2(__float_as_int(g), first ? c : -1);
  }
  loss = wave_add(loss) * a.t * a.t;
  if (lane == 0) {
    a.loss[row] = norm == 0.0f && !bad ? 0.0f : (coef != coef ? coef : loss);
    a.lse[row] = static_cast<float>(kLn2 * (l2 + m * k));
    *reinterpret_cast<v4i*>(state) = v4i{m, __float_as_int(static_cast<float>(l2)), __float_as_int(coef), 0};
  }
}

// the targets' gradients into a piece of the softmax
__global__ __launch_bounds__(256) void vocab_targets_kernel(const int32_t* __restrict__ state, int rows, int top, long long first, int classes,
                                                            _Float16* __restrict__ g, long long pitch) {
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= static_cast<long long>(rows) * top) return;
  const long long row = at / top;
  const int32_t* const s = state + row * vocab_state_words(top) + 4 + 2 * (at - row * top);
  const long long c = s[1] - first;
  if (s[1] >= 0 && c >= 0 && c < classes) g[row * pitch + c] = static_cast<_Float16>(ldexpf(__int_as_float(s[0]), kGradExponent));
}

// ---- host ------------------------------------------------------------------------------------------------------------
struct Matrix {      // as the caller has it, or a copy with rows of a multiple of 16
  const int8_t* p;
  long long pitch;
  long long rows;
  int row_bytes;
};
// The products read 16 bytes at a time from addresses that are multiples of four.  Activations want zeros behind their features where these are no
// multiple of 16: the weights' row ends then do not matter.
bool off_four(const Matrix& m) { return ((reinterpret_cast<uintptr_t>(m.p) | static_cast<uintptr_t>(m.pitch)) & 3) != 0; }
bool copy_activations(const Matrix& m, int features) { return off_four(m) || features % 16 != 0; }
bool copy_weights(const Matrix& m, int features) { return off_four(m) || features % 4 != 0; }

struct Layout {
  size_t bytes = 0;
  size_t take(long long n) {
    const size_t at = bytes;
    bytes += static_cast<size_t>(round_up(n, 256));
    return at;
  }
};

struct ForwardPlan {
  size_t a, w, part, bytes;
  bool copy_a, copy_w;
  VocabTile tile;
  int tiles;
};
ForwardPlan forward_plan(const Matrix& a, const Matrix& w, int features) {
  ForwardPlan p{};
  Layout l;
  const long long row = round_up(features, 16);
  p.copy_a = copy_activations(a, features);
  p.copy_w = copy_weights(w, features);
  p.a = l.take(p.copy_a ? a.rows * row : 0);
  p.w = l.take(p.copy_w ? w.rows * row : 0);
  p.tile = vocab_logits_tile(static_cast<int>(a.rows), features, static_cast<int>(w.rows));
  p.tiles = vocab_stats_tiles(p.tile, static_cast<int>(w.rows));
  p.part = l.take(a.rows * p.tiles * 8);
  p.bytes = l.bytes;
  return p;
}

struct BackwardPlan {
  size_t a, w, wide_a, wide_w, grad, part_a, part_w, exponent, bytes;
  bool copy_a, copy_w;
  long long piece, pitch16, part_pitch;   // classes at a time; values of a 16-bit row; values of a partial sum's row
  VocabTile tile;
  int slices_a, steps_a, slices_w, steps_w;
  bool parts_a, parts_w;
};
BackwardPlan backward_plan(const Matrix& a, const Matrix& w, int features, bool f32) {
  BackwardPlan p{};
  Layout l;
  const long long row = round_up(features, 16);
  p.copy_a = copy_activations(a, features);
  p.copy_w = copy_weights(w, features);
  p.pitch16 = row;
  p.part_pitch = round_up(features, 4);
  long long piece = kPieceGrad / a.rows;
  if (a.rows > 32 && piece > kPieceWide / features) piece = kPieceWide / features;
  if (piece < kPieceLeast) piece = kPieceLeast;
  if (piece > kPieceMost) piece = kPieceMost;
  piece = piece / 256 * 256;
  if (piece > round_up(w.rows, 8)) piece = round_up(w.rows, 8);
  p.piece = piece;
  p.tile = vocab_sums_plan(static_cast<int>(a.rows), features, static_cast<int>(piece), &p.slices_a, &p.steps_a, &p.slices_w, &p.steps_w);
  p.parts_a = f32 || p.slices_a > 1 || piece < w.rows;      // float32 results leave by way of the join
  p.parts_w = f32 || p.slices_w > 1;
  p.a = l.take(p.copy_a ? a.rows * row : 0);
  p.w = l.take(p.copy_w ? w.rows * row : 0);
  p.wide_a = l.take(a.rows * p.pitch16 * 2);
  p.wide_w = l.take(vocab_sums_wants_wide_weights(p.tile) ? piece * p.pitch16 * 2 : 0);
  p.grad = l.take(a.rows * piece * 2);
  p.part_a = l.take(p.parts_a ? p.slices_a * a.rows * p.part_pitch * 4 : 0);
  p.part_w = l.take(p.parts_w ? p.slices_w * piece * p.part_pitch * 4 : 0);
  p.exponent = l.take(4);
  p.bytes = l.bytes;
  return p;
}

// copies what cannot be read in place, and points a and w at the copies
int pad_rows(Matrix* a, bool copy_a, int8_t* to_a, Matrix* w, bool copy_w, int8_t* to_w, int features, hipStream_t stream) {
  if (!copy_a && !copy_w) return NITI_OK;
  const auto pad = [features](const Matrix& m, bool copy, int8_t* to) {
    return VocabPad{m.p, m.pitch, to, m.rows, copy ? static_cast<int>((m.rows * ((features + 15) / 16) + 255) / 256) : 0};
  };
  const VocabPad pa = pad(*a, copy_a, to_a), pw = pad(*w, copy_w, to_w);
  if (const int rc = check_grid(static_cast<long long>(pa.blocks) + pw.blocks, 256, "vocab_pad")) return rc;
  hipLaunchKernelGGL(vocab_pad_kernel, dim3(static_cast<unsigned>(pa.blocks) + static_cast<unsigned>(pw.blocks)), dim3(256), 0, stream, pa, pw, features);
  if (copy_a) *a = Matrix{to_a, round_up(features, 16), a->rows, static_cast<int>(round_up(features, 16))};
  if (copy_w) *w = Matrix{to_w, round_up(features, 16), w->rows, static_cast<int>(round_up(features, 16))};
  return check_launch("vocab_pad");
}
VocabOperand bytes_operand(const Matrix& m) {
  return VocabOperand{m.p, m.pitch, static_cast<int>(m.rows), m.row_bytes};
}

int check_operands(const char* who, const int8_t* act, long long act_pitch, const int8_t* w, long long w_pitch, const int32_t* exp_a, const int32_t* exp_w,
                   int rows, int features, int classes, int top) {
  if (act == nullptr || w == nullptr || exp_a == nullptr || exp_w == nullptr) return fail(NITI_ERR_INVALID_ARG, "%s: null pointer", who);
  if (rows <= 0 || features <= 0 || classes <= 0 || top <= 0)
    return fail(NITI_ERR_INVALID_ARG, "%s: rows=%d features=%d classes=%d top=%d", who, rows, features, classes, top);
  if (act_pitch < features || w_pitch < features) return fail(NITI_ERR_INVALID_ARG, "%s: rows of %lld and %lld bytes hold no %d features", who, act_pitch, w_pitch, features);
  if (features > kMaxFeatures) return fail(NITI_ERR_UNSUPPORTED, "%s: %d features (at most %d)", who, features, kMaxFeatures);
  if (rows > kMaxRows) return fail(NITI_ERR_UNSUPPORTED, "%s: %d rows (at most %d)", who, rows, kMaxRows);
  if (act_pitch >= (1LL << 22) || w_pitch >= (1LL << 22)) return fail(NITI_ERR_UNSUPPORTED, "%s: rows 4 MiB or more apart", who);
  if (top > kVocabTopMost) return fail(NITI_ERR_UNSUPPORTED, "%s: lists of %d (at most %d)", who, top, kVocabTopMost);
  return NITI_OK;
}

int forward(const char* who, const int8_t* act, long long act_pitch, const int8_t* w, long long w_pitch, const int32_t* exp_a, const int32_t* exp_w, int rows,
            int features, int classes, const void* value, int value_type, const void* index, int index_bytes, long long ignored, int top, float t, float* loss,
            float* lse, int32_t* state, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check_operands(who, act, act_pitch, w, w_pitch, exp_a, exp_w, rows, features, classes, top)) return rc;
  if (index == nullptr || loss == nullptr || lse == nullptr || state == nullptr) return fail(NITI_ERR_INVALID_ARG, "%s: null pointer", who);
  if (index_bytes != 4 && index_bytes != 8) return fail(NITI_ERR_INVALID_ARG, "%s: classes of %d bytes (4 or 8)", who, index_bytes);
  if (!aligned16(state)) return fail(NITI_ERR_INVALID_ARG, "%s: state not 16-byte aligned", who);
  Matrix a{act, act_pitch, rows, features}, b{w, w_pitch, classes, features};
  const ForwardPlan p = forward_plan(a, b, features);
  if (workspace == nullptr || workspace_bytes < p.bytes || !aligned16(workspace))
    return fail(NITI_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, p.bytes, workspace_bytes);
  char* const ws = static_cast<char*>(workspace);
  if (const int rc = pad_rows(&a, p.copy_a, reinterpret_cast<int8_t*>(ws + p.a), &b, p.copy_w, reinterpret_cast<int8_t*>(ws + p.w), features, stream)) return rc;
  int2* const part = reinterpret_cast<int2*>(ws + p.part);
  const VocabLogits l{bytes_operand(b), bytes_operand(a), classes, rows, features, exp_a, exp_w, 1.0f / t};
  const VocabTargets targets{index, index_bytes, value != nullptr ? 1 : 0, ignored, top, state};
  if (const int rc = launch_vocab_stats(p.tile, l, VocabStats{part, p.tiles}, targets, stream)) return rc;
  const VocabRows r{part, p.tiles, rows, classes, exp_a, exp_w, t, targets, value, value_type, loss, lse, state};
  hipLaunchKernelGGL(vocab_rows_kernel, dim3(rows), dim3(64), 8 * top, stream, r);
  return check_launch(who);
}

// d_act, d_w: bfloat16, or float32 by f32
int backward(const int8_t* act, long long act_pitch, const int8_t* w, long long w_pitch, const int32_t* exp_a, const int32_t* exp_w, int rows, int features,
             int classes, int top, float temperature, const int32_t* state, const float* weight, int weights, void* d_act, void* d_w, bool f32, void* workspace,
             size_t workspace_bytes, hipStream_t st) {
  const char* const who = "vocab_backward";
  const auto out16 = [f32](void* p, long long at) { return f32 ? nullptr : static_cast<uint16_t*>(p) + at; };
  const auto out32 = [f32](void* p, long long at) { return f32 ? static_cast<float*>(p) + at : nullptr; };
  if (const int rc = check_operands(who, act, act_pitch, w, w_pitch, exp_a, exp_w, rows, features, classes, top)) return rc;
  if (state == nullptr || d_act == nullptr || d_w == nullptr) return fail(NITI_ERR_INVALID_ARG, "%s: null pointer", who);
  if (weight != nullptr && weights != 1 && weights != rows) return fail(NITI_ERR_INVALID_ARG, "%s: %d weights for %d rows", who, weights, rows);
  if (!(temperature > 0.0f) || !isfinite(temperature)) return fail(NITI_ERR_INVALID_ARG, "%s: temperature %g", who, static_cast<double>(temperature));
  if (!aligned16(state) || !aligned16(d_act) || !aligned16(d_w)) return fail(NITI_ERR_INVALID_ARG, "%s: state or result not 16-byte aligned", who);
  Matrix a{act, act_pitch, rows, features}, b{w, w_pitch, classes, features};
  const BackwardPlan p = backward_plan(a, b, features, f32);
  if (const int rc = check_grid((static_cast<long long>(rows) * ((features + 3) / 4) + 255) / 256, 256, "vocab_join")) return rc;      // before anything runs
  if (workspace == nullptr || workspace_bytes < p.bytes || !aligned16(workspace))
    return fail(NITI_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, p.bytes, workspace_bytes);
  char* const ws = static_cast<char*>(workspace);
  if (const int rc = pad_rows(&a, p.copy_a, reinterpret_cast<int8_t*>(ws + p.a), &b, p.copy_w, reinterpret_cast<int8_t*>(ws + p.w), features, st)) return rc;
  _Float16* const wide_a = reinterpret_cast<_Float16*>(ws + p.wide_a);
  _Float16* const wide_w = reinterpret_cast<_Float16*>(ws + p.wide_w);
  const bool wide_weights = vocab_sums_wants_wide_weights(p.tile);
  _Float16* const grad = reinterpret_cast<_Float16*>(ws + p.grad);
  int32_t* const exponent = reinterpret_cast<int32_t*>(ws + p.exponent);
  // weights of the rows go into the activations' 16-bit copy (their sum over the rows is one product); one weight for all into the result
  const bool each = weight != nullptr && weights == rows && rows > 1;
  const auto widen_blocks = [features](long long n) {      // 512 lanes of sixteen values, at most two workgroups per unit
    const long long blocks = (n * round_up(features, 16) / 16 + 511) / 512;
    return static_cast<int>(blocks < 512 ? blocks : 512);
  };

  for (long long first = 0; first < classes; first += p.piece) {
    const int here = static_cast<int>(classes - first < p.piece ? classes - first : p.piece);
    const Matrix piece{b.p + first * b.pitch, b.pitch, here, b.row_bytes};
    const VocabLogits l{bytes_operand(piece), bytes_operand(a), here, rows, features, exp_a, exp_w, 1.0f / temperature};
    const VocabTile tile = vocab_logits_tile(rows, features, here);
    const bool targets = vocab_grad_writes_targets(tile, top);
    const VocabWiden widen_a{a.p, a.pitch, a.row_bytes, wide_a, p.pitch16, rows, features, each ? weight : nullptr, exponent, first == 0 ? widen_blocks(rows) : 0};
    const VocabWiden widen_w{piece.p, piece.pitch, piece.row_bytes, wide_w, p.pitch16, here, features, nullptr, nullptr, wide_weights ? widen_blocks(here) : 0};
    if (const int rc = launch_vocab_grad(tile, l, VocabGrad{state, vocab_state_words(top), targets ? top : 0, first, grad, p.piece, widen_a, widen_w}, st)) return rc;
    if (!targets) {
      const long long places = static_cast<long long>(rows) * top;
      if (const int rc = check_grid((places + 255) / 256, 256, "vocab_targets")) return rc;
      hipLaunchKernelGGL(vocab_targets_kernel, dim3(static_cast<unsigned>((places + 255) / 256)), dim3(256), 0, st, state, rows, top, first, here, grad, p.piece);
      if (const int rc = check_launch(who)) return rc;
    }

    const int stages = (here + 63) / 64;
    VocabSums sa{wide_weights ? VocabOperand{wide_w, p.pitch16 * 2, here, static_cast<int>(p.pitch16 * 2)}
                              : VocabOperand{piece.p, piece.pitch, here, piece.row_bytes},
                 VocabOperand{grad, p.piece * 2, rows, static_cast<int>(round_up(here, 8) * 2)}, features, rows, here, (stages + p.steps_a - 1) / p.steps_a, p.steps_a,
                 p.parts_a ? reinterpret_cast<float*>(ws + p.part_a) : nullptr, p.part_pitch, first > 0 ? 1 : 0, out16(d_act, 0), out32(d_act, 0), temperature, exp_w, -kGradExponent, nullptr,
                 weight, weights};
    const VocabSums sw{VocabOperand{wide_a, p.pitch16 * 2, rows, static_cast<int>(p.pitch16 * 2)}, VocabOperand{grad, p.piece * 2, rows, static_cast<int>(p.piece * 2)},
                       features, here, rows, p.slices_w, p.steps_w, p.parts_w ? reinterpret_cast<float*>(ws + p.part_w) : nullptr, p.part_pitch, 0,
                       out16(d_w, first * features), out32(d_w, first * features), temperature, exp_a, -kGradExponent - (each ? kRowExponent : 0), each ? exponent : nullptr, each ? nullptr : weight, 1};
    if (const int rc = launch_vocab_sums(p.tile, sa, sw, st)) return rc;
    const bool join_a = p.parts_a && first + p.piece >= classes;
    sa.slices = p.slices_a;
    if (join_a || p.parts_w) {
      if (const int rc = launch_vocab_join(join_a ? &sa : nullptr, p.parts_w ? &sw : nullptr, st)) return rc;
    }
  }
  return NITI_OK;
}

}  // namespace
}  // namespace niti

using namespace niti;

extern "C" size_t niti_vocab_state_words(int top) { return top > 0 ? static_cast<size_t>(vocab_state_words(top)) : 0; }

extern "C" size_t niti_vocab_forward_workspace(const int8_t* act, int64_t act_pitch, const int8_t* w, int64_t w_pitch, int rows, int features, int classes) {
  if (rows <= 0 || features <= 0 || classes <= 0) return 0;
  return forward_plan(Matrix{act, act_pitch, rows, features}, Matrix{w, w_pitch, classes, features}, features).bytes;
}

extern "C" size_t niti_vocab_backward_workspace(const int8_t* act, int64_t act_pitch, const int8_t* w, int64_t w_pitch, int rows, int features, int classes) {
  if (rows <= 0 || features <= 0 || classes <= 0) return 0;
  return backward_plan(Matrix{act, act_pitch, rows, features}, Matrix{w, w_pitch, classes, features}, features, false).bytes;
}

extern "C" size_t niti_vocab_backward_f32_workspace(const int8_t* act, int64_t act_pitch, const int8_t* w, int64_t w_pitch, int rows, int features, int classes) {
  if (rows <= 0 || features <= 0 || classes <= 0) return 0;
  return backward_plan(Matrix{act, act_pitch, rows, features}, Matrix{w, w_pitch, classes, features}, features, true).bytes;
}

extern "C" int niti_vocab_plan(int rows, int features, int classes, int* plan) {
  clear_error();
  if (plan == nullptr || rows <= 0 || features <= 0 || classes <= 0) return fail(NITI_ERR_INVALID_ARG, "vocab_plan: rows=%d features=%d classes=%d", rows, features, classes);
  const BackwardPlan p = backward_plan(Matrix{nullptr, features, rows, features}, Matrix{nullptr, features, classes, features}, features, false);
  plan[0] = vocab_logits_tile(rows, features, classes);
  plan[1] = vocab_logits_tile(rows, features, static_cast<int>(p.piece < classes ? p.piece : classes));
  plan[2] = p.tile;
  plan[3] = static_cast<int>(p.piece);
  plan[4] = p.slices_a;
  plan[5] = p.slices_w;
  return NITI_OK;
}

extern "C" int niti_vocab_entropy_i8(const int8_t* act, int64_t act_pitch, const int8_t* w, int64_t w_pitch, const int32_t* exp_a, const int32_t* exp_w, int rows,
                                     int features, int classes, const void* target, int target_bytes, int64_t ignored, float* loss, float* lse, int32_t* state,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  return forward("vocab_entropy", act, act_pitch, w, w_pitch, exp_a, exp_w, rows, features, classes, nullptr, 0, target, target_bytes, ignored, 1, 1.0f, loss, lse,
                 state, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int niti_vocab_distill_i8(const int8_t* act, int64_t act_pitch, const int8_t* w, int64_t w_pitch, const int32_t* exp_a, const int32_t* exp_w, int rows,
                                     int features, int classes, const void* top_value, int value_type, const void* top_class, int class_bytes, int top,
                                     float temperature, float* loss, float* lse, int32_t* state, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (top_value == nullptr) return fail(NITI_ERR_INVALID_ARG, "vocab_distill: null pointer");
  if (value_type != NITI_F32 && value_type != NITI_BF16 && value_type != NITI_F16) return fail(NITI_ERR_INVALID_ARG, "vocab_distill: value_type=%d", value_type);
  if (!(temperature > 0.0f) || !isfinite(temperature)) return fail(NITI_ERR_INVALID_ARG, "vocab_distill: temperature %g", static_cast<double>(temperature));
  return forward("vocab_distill", act, act_pitch, w, w_pitch, exp_a, exp_w, rows, features, classes, top_value, value_type, top_class, class_bytes, -1, top, temperature,
                 loss, lse, state, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int niti_vocab_backward_i8(const int8_t* act, int64_t act_pitch, const int8_t* w, int64_t w_pitch, const int32_t* exp_a, const int32_t* exp_w, int rows,
                                      int features, int classes, int top, float temperature, const int32_t* state, const float* weight, int weights,
                                      uint16_t* d_act, uint16_t* d_w, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  return backward(act, act_pitch, w, w_pitch, exp_a, exp_w, rows, features, classes, top, temperature, state, weight, weights, d_act, d_w, false, workspace,
                  workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int niti_vocab_backward_i8_f32(const int8_t* act, int64_t act_pitch, const int8_t* w, int64_t w_pitch, const int32_t* exp_a, const int32_t* exp_w, int rows,
                                          int features, int classes, int top, float temperature, const int32_t* state, const float* weight, int weights,
                                          float* d_act, float* d_w, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  return backward(act, act_pitch, w, w_pitch, exp_a, exp_w, rows, features, classes, top, temperature, state, weight, weights, d_act, d_w, true, workspace,
                  workspace_bytes, static_cast<hipStream_t>(stream));
}
