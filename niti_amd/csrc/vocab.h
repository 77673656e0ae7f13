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

typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// p and g lie in [-1, 1]; as 16-bit floats they are kept times 2^15: eleven significant bits down to 2^-29, where bfloat16 has eight
constexpr int kGradExponent = 15;
// rows of the second product's left operand: activation times row weight over the largest row weight's power of two, times 2^8
constexpr int kRowExponent = 8;
constexpr int kVocabTopMost = 1024;      // places of a teacher's list (one row's are kept in LDS)
constexpr int kVocabClassTile = 256;     // classes that leave one (maximum, sum) pair of a row

// What a forward pass leaves of a row: m, L (float), the sum of the targets' weights (float: 1; 0, nothing to learn from; NaN,
// undefined), a word of nothing, then for each of its `top` places g / T (float) and the class, -1 where there is none or an earlier place
// has named it.  Rows start on 16 bytes.
inline __host__ __device__ long long vocab_state_words(int top) { return 4 + (2LL * top + 3) / 4 * 4; }

// One operand of a product tile: rows of `pitch` bytes, 16-byte aligned.
//   reduction index fast: `rows` rows of `row_bytes` bytes (a multiple of 16)
//   reduction index slow: `rows` steps of the reduction, tile columns along the row
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

struct VocabStats {          // (max, sum of 2^((s - max) k)) of each row over each kVocabClassTile classes
  int2* part;                // [rows][tiles]
  int tiles;
};

struct VocabGrad {           // sum_j q_j p, times 2^kGradExponent, of the classes of a piece
  const int32_t* state;      // [rows][state_words]
  long long state_words;
  _Float16* g;               // [rows][pitch], zero between the piece's last class and the next multiple of eight
  long long pitch;
};

struct VocabSums {           // out[j][i] = sum_k x[i][k] y[j][k] in float
  VocabOperand x, y;
  int ni, nj, nk;
  int slices, steps;         // reduction cut in `slices` parts of `steps` stages of 64
  float* part;               // [slices][nj][part_pitch]; null: written to out at once
  long long part_pitch;
  int accumulate;            // add to what part holds
  uint16_t* out;             // bfloat16 [nj][ni]
  // scale of the result: T 2^(exponent) weight
  float t;
  const int32_t* exponent;
  int bias;
  const int32_t* exponent2;  // may be null
  const float* weight;       // per j; null: 1.  weight_n == 1: the same for all
  int weight_n;
};

int launch_vocab_stats(const VocabLogits& l, const VocabStats& s, hipStream_t stream);
int launch_vocab_grad(const VocabLogits& l, const VocabGrad& g, hipStream_t stream);
int launch_vocab_sums(const VocabSums& s, bool y_slow, hipStream_t stream);   // x's reduction index is the slow one, y's may be
int launch_vocab_join(const VocabSums& s, hipStream_t stream);
void vocab_sums_plan(int ni, int nj, int nk, int* slices, int* steps);

}  // namespace niti
