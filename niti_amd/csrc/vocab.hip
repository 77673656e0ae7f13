// Products of the losses over a large vocabulary (vocab.h): the logits' statistics, a piece of their gradient, and the sums of the
// two gradients behind it.  One tile product serves all three.
//
// Tile: TI x TJ results of sum_k x[i][k] y[j][k]; lane l of a wavefront holds for each 16 x 16 block column j = l % 16 and the rows
// i = 4 (l / 16) .. + 4 (v_mfma_i32_16x16x64_i8 or v_mfma_f32_16x16x32_f16, 64 bytes of the reduction each).  A stage is 128 bytes of
// the reduction, two buffers, filled by buffer_load ... lds while the other one is multiplied.  An operand whose reduction
// index is fast is staged as whole 128-byte lines, 16-byte pieces XOR-swizzled by row / 2 so that the 16 rows a fragment read takes lie in
// different banks; one whose reduction index is slow (16-bit values only) lies as stored, 64 steps of TI or TJ columns, and is
// transposed by ds_read_b64_tr_b16, its 32-byte pieces XOR-swizzled by the step.
#include "lds_asm.h"
#include "vocab.h"

namespace niti {
namespace {

constexpr int kFar = static_cast<int>(0x80000000u);   // beyond every buffer: reads as zero
constexpr int kStageBytes = 128;                      // of the reduction

template <int TI_, int TJ_, int WI_, int WJ_>
struct Tile {
  static constexpr int TI = TI_, TJ = TJ_, WI = WI_, WJ = WJ_;
  static constexpr int kWaves = WI * WJ, kThreads = 64 * kWaves;
  static constexpr int BI = TI / WI / 16, BJ = TJ / WJ / 16;   // 16 x 16 blocks of a wavefront
  static constexpr int kLds = 2 * (TI + TJ) * kStageBytes;
  // workgroups per unit that the registers are cut for: two wavefronts per SIMD at least, so that all sums are ordinary registers
  static constexpr int kPerUnit = kWaves >= 8 ? 1 : 8 / kWaves;
};
typedef Tile<256, 256, 2, 4> TileLarge;
typedef Tile<128, 128, 2, 2> TileMiddle;
typedef Tile<256, 32, 8, 1> TileFew;

// 16-lane groups: lane i of a group names 8 bytes of a 4 x 16 block of 16-bit values (row i / 4, columns 4 (i % 4) .. + 4) and receives
// column i of it
template <int OFF>
__device__ inline v2i lds_read_tr16(unsigned addr) {
  v2i r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
  return r;
}

__device__ inline void tile_sync() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One operand's way from memory to fragments: R rows (or columns, where the reduction index is slow).
template <int R, bool kSlow, int kWaves>
struct Source {
  static constexpr int kInstructions = R * kStageBytes / 1024;              // of a stage
  static constexpr int kLoads = (kInstructions + kWaves - 1) / kWaves;      // of a wavefront, 16 bytes per lane each
  static constexpr int kRowBytes = kSlow ? 2 * R : kStageBytes;
  static constexpr int kRowsPerLoad = 1024 / kRowBytes;
  static constexpr int kPieces = kRowBytes / 16;
  static_assert(kInstructions % kWaves == 0 || kInstructions < kWaves, "whole wavefronts");

  const char* base;
  long long left;        // bytes from base to the end of the matrix
  long long advance;     // per stage
  int fast_left;         // bytes of the reduction left in a row (reduction fast)
  int voff[kLoads];
  int piece;

  // slow position of a reduction step within its stage that its 32-byte pieces are swizzled by: the eight steps that 32 lanes read
  // at once (four of each 16-lane group, groups eight steps apart) differ in it
  static __device__ int turn(int k) { return ((k & 3) | (((k >> 3) & 1) << 2)) & (R / 16 - 1); }

  // first: first row (fast) or column (slow) of the tile; k0: first reduction step in stages; k_end: end of the reduction's range in bytes (fast)
  // or steps (slow)
  __device__ void init(const VocabOperand& o, int first, int k0, int k_end) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const char* const p = static_cast<const char*>(o.p);
    if (kSlow) {
      const long long skip = static_cast<long long>(k0) * 64 * o.pitch + 2LL * first;
      base = p + skip;
      left = static_cast<long long>(k_end) * o.pitch - skip;
      advance = 64 * o.pitch;
      fast_left = 0;
      piece = 0;
    } else {
      const long long skip = first * o.pitch + static_cast<long long>(k0) * kStageBytes;
      base = p + skip;
      left = (o.rows - 1) * o.pitch + o.row_bytes - skip;
      advance = kStageBytes;
      fast_left = k_end - k0 * kStageBytes;
    }
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int row = (q * kWaves + wave) * kRowsPerLoad + lane / kPieces;
      const int slot = lane % kPieces;
      const int c = kSlow ? slot ^ (2 * turn(row)) : slot ^ ((row >> 1) & 7);
      if (!kSlow) piece = c * 16;       // the same for every q: a load's rows are a multiple of 16 apart
      voff[q] = static_cast<int>(row * o.pitch) + c * 16;
    }
  }

  // the stage that load() fetches instructions of; next() moves on
  __device__ __amdgpu_buffer_rsrc_t stage() const {
    const int n = left <= 0 ? 0 : (left > 0x7fffffffLL ? 0x7fffffff : static_cast<int>(left));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, n, 0x00020000);
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned lds, int q) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (kInstructions >= kWaves || wave < kInstructions)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, NITI_LDS_AT(lds + (q * kWaves + wave) * 1024), 16, kSlow || piece < fast_left ? voff[q] : kFar, 0, 0, 0);
  }
  __device__ void next() {
    base += advance;
    left -= advance;
    fast_left -= kStageBytes;
  }
};

// Fragment reads of B blocks of 16 rows / columns, starting at block `first` of the operand's stages at LDS address `lds`.
template <int R, int B, bool kSlow>
struct Fragments {
  unsigned addr[kSlow ? B : 2];
  v2i lo[2][kSlow ? B : 1], hi[2][kSlow ? B : 1];     // of the two halves of a stage
  v4i whole[2][kSlow ? 1 : B];

  __device__ void init(unsigned lds, int first) {
    const int lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    if constexpr (kSlow) {
      const int t = ((i >> 2) | ((g & 1) << 2)) & (R / 16 - 1);      // Source::turn of steps 8 g + i / 4 (+ 4, + 32)
#pragma unroll
      for (int b = 0; b < B; ++b) addr[b] = lds + (8 * g + (i >> 2)) * (2 * R) + (((first + b) ^ t) << 5) + (i & 3) * 8;
    } else {
      addr[0] = lds + (first * 16 + i) * kStageBytes + ((g ^ (i >> 1)) << 4);
      addr[1] = addr[0] ^ 64;
    }
  }
  __device__ void other_buffer(int step) {
#pragma unroll
    for (int b = 0; b < (kSlow ? B : 2); ++b) addr[b] += step;
  }
  template <int SUB, int BLK>
  __device__ void read() {
    if constexpr (kSlow) {
      lo[SUB][BLK] = lds_read_tr16<SUB * 64 * R>(addr[BLK]);
      hi[SUB][BLK] = lds_read_tr16<SUB * 64 * R + 8 * R>(addr[BLK]);
    } else {
      whole[SUB][BLK] = lds_read_b128_at<BLK * 16 * kStageBytes>(addr[SUB]);
    }
  }
  // behind a settle: the reads of half SUB are in their registers
  template <int SUB>
  __device__ void landed() {
    if constexpr (kSlow) {
#pragma unroll
      for (int b = 0; b < B; ++b) asm volatile("" : "+v"(lo[SUB][b]), "+v"(hi[SUB][b]));
    } else {
#pragma unroll
      for (int b = 0; b < B; ++b) asm volatile("" : "+v"(whole[SUB][b]));
    }
  }
  template <int SUB, int BLK>
  __device__ v4i get() const {
    if constexpr (kSlow) return v4i{lo[SUB][BLK][0], lo[SUB][BLK][1], hi[SUB][BLK][0], hi[SUB][BLK][1]};
    else return whole[SUB][BLK];
  }
};

__device__ inline v4i multiply(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
__device__ inline v4f multiply(v4i a, v4i b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Main loop.  Half a stage's fragments are read while the other half is multiplied, and the barrier lies between the halves: behind it
// the next stage's first half is requested in front of the second half's products, and the loads of the stage after that go out, so no
// product waits for the reads behind a barrier.  The fragments carried into the next turn have landed by the end of one.
template <class T, bool kXSlow, bool kYSlow, class Acc>
struct Product {
  Source<T::TI, kXSlow, T::kWaves> sx;
  Source<T::TJ, kYSlow, T::kWaves> sy;
  Fragments<T::TI, T::BI, kXSlow> fx;
  Fragments<T::TJ, T::BJ, kYSlow> fy;
  Acc acc[T::BI][T::BJ];
  unsigned ldsx, ldsy;

  static constexpr int kLoadsX = decltype(sx)::kLoads, kLoadsY = decltype(sy)::kLoads;

  // instruction q of a stage's loads into buffer buf
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rx, __amdgpu_buffer_rsrc_t ry, int buf, int q) const {
    if (q < kLoadsX) sx.load(rx, ldsx + buf * T::TI * kStageBytes, q);
    else sy.load(ry, ldsy + buf * T::TJ * kStageBytes, q - kLoadsX);
  }
  __device__ void issue(int buf) {
    const __amdgpu_buffer_rsrc_t rx = sx.stage(), ry = sy.stage();
    static_for<kLoadsX + kLoadsY>([&](auto q) { load(rx, ry, buf, decltype(q)::value); });
    sx.next();
    sy.next();
  }
  // Products of half SUB; half NEXT is read in between, and where kLoad the next stage but one goes out into buffer buf, spread over the
  // products: a unit's loads pass at 64 bytes a clock, and a wavefront waits at a load that finds the queue full
  template <int SUB, int NEXT, bool kLoad>
  __device__ void half(int buf) {
    const __amdgpu_buffer_rsrc_t rx = sx.stage(), ry = sy.stage();
    static_for<T::BI>([&](auto i) {
      constexpr int I = decltype(i)::value;
      if constexpr (I < T::BJ) fy.template read<NEXT, I>();
      fx.template read<NEXT, I>();
     __builtin_amdgcn_s_setprio(1);  static_for<T::BJ>([&](auto j) {
        constexpr int J = decltype(j)::value;
        acc[I][J] = multiply(fx.template get<SUB, I>(), fy.template get<SUB, J>(), acc[I][J]);
      });
      if constexpr (kLoad) {
        constexpr int kAll = kLoadsX + kLoadsY, kFrom = I * kAll / T::BI, kTo = (I + 1) * kAll / T::BI;
        static_for<kTo - kFrom>([&](auto q) { load(rx, ry, buf, kFrom + decltype(q)::value); });
      }
    __builtin_amdgcn_s_setprio(0);  __builtin_amdgcn_sched_barrier(0);      // keeps reads, products and loads in this order
    });
    if constexpr (kLoad) {
      sx.next();
      sy.next();
    }
    lds_settle<0>();
    fx.template landed<NEXT>();
    fy.template landed<NEXT>();
  }

  // x, y: operands; i0, j0: the tile's corner; range of the reduction: stages k0 .. k0 + n, ending at x_end and y_end (bytes or steps)
  __device__ void run(const VocabOperand& x, const VocabOperand& y, int i0, int j0, int k0, int n, int x_end, int y_end, char* smem) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ldsx = lds_addr(smem);
    ldsy = ldsx + 2 * T::TI * kStageBytes;
    sx.init(x, i0, k0, x_end);
    sy.init(y, j0, k0, y_end);
    fx.init(ldsx, (wave / T::WJ) * T::BI);
    fy.init(ldsy, (wave % T::WJ) * T::BJ);
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int j = 0; j < T::BJ; ++j) acc[i][j] = Acc{0, 0, 0, 0};
    // loads of the two stages behind the last are issued like the others: they are out of range, and what they clear is not multiplied
    issue(0);
    issue(1);
    constexpr int kLeast = (Source<T::TI, kXSlow, T::kWaves>::kInstructions + Source<T::TJ, kYSlow, T::kWaves>::kInstructions) / T::kWaves;   // loads per stage
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeast) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    static_for<T::BJ>([&](auto j) { fy.template read<0, decltype(j)::value>(); });
    static_for<T::BI>([&](auto i) { fx.template read<0, decltype(i)::value>(); });
    lds_settle<0>();
    fx.template landed<0>();
    fy.template landed<0>();
    int buf = 0;
    for (int s = 0; s < n; ++s) {
      half<0, 1, false>(buf);
      tile_sync();          // the next stage has landed, and this one's buffer has been read by every wavefront
      const int step = buf == 0 ? 1 : -1;
      fx.other_buffer(step * T::TI * kStageBytes);
      fy.other_buffer(step * T::TJ * kStageBytes);
      half<1, 0, true>(buf);
      buf ^= 1;
    }
    tile_sync();            // the buffers are free
  }
};

// Workgroup -> tile: a die (every eighth workgroup) takes a run of tiles, and a run goes down `kRows` tile rows before the next column,
// so that the tiles in flight on a die share their operands in its L2.
__device__ inline void tile_of(int block, int ti, int tj, int* i, int* j) {
  const int total = ti * tj;
  const int die = block & 7, per = total >> 3, extra = total & 7;
  const int t = die * per + (die < extra ? die : extra) + (block >> 3);
  constexpr int kRows = 8;
  const int band = t / (kRows * tj), r = t - band * kRows * tj;
  const int rows = ti - band * kRows < kRows ? ti - band * kRows : kRows;
  *j = r / rows;
  *i = band * kRows + r - *j * rows;
}

// k of vocab.h, finite: an overflow would make 0 k a NaN where it stands for a difference of nothing
__device__ inline float exp2_scale(const VocabLogits& l) {
  const float k = ldexpf(1.44269504088896340736f * l.inv_t, *l.exp_a + *l.exp_w);
  return fminf(k, 3.402823466e38f);
}

template <class T>
__global__ __launch_bounds__(T::kThreads, T::kPerUnit) void vocab_stats_kernel(const VocabLogits l, const VocabStats st) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int bi, bj;
  tile_of(blockIdx.x, (l.classes + T::TI - 1) / T::TI, (l.rows + T::TJ - 1) / T::TJ, &bi, &bj);
  const int i0 = bi * T::TI, j0 = bj * T::TJ;
  Product<T, false, false, v4i> p;
  p.run(l.w, l.a, i0, j0, 0, (l.features + kStageBytes - 1) / kStageBytes, l.w.row_bytes, l.a.row_bytes, smem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / T::WJ, wj = wave % T::WJ;
  const float k = exp2_scale(l);
  int2* const park = reinterpret_cast<int2*>(smem);   // [WI][TJ]
  const int v0 = i0 + wi * T::BI * 16 + 4 * (lane >> 4);
  const bool whole = i0 + T::TI <= l.classes;
#pragma unroll
  for (int j = 0; j < T::BJ; ++j) {
    int m = -2147483647 - 1;
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (whole || v0 + i * 16 + r < l.classes) m = max(m, p.acc[i][j][r]);
    m = max(m, __shfl_xor(m, 16, 64));
    m = max(m, __shfl_xor(m, 32, 64));
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (whole || v0 + i * 16 + r < l.classes) sum += __builtin_amdgcn_exp2f(static_cast<float>(p.acc[i][j][r] - m) * k);
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 16) park[wi * T::TJ + (wj * T::BJ + j) * 16 + lane] = make_int2(m, __float_as_int(sum));
  }
  __syncthreads();
  // one pair of each row for every kVocabClassTile classes
  constexpr int kGroups = T::TI < kVocabClassTile ? 1 : T::TI / kVocabClassTile;
  static_assert(kGroups == 1, "a tile leaves one pair");
  for (int j = threadIdx.x; j < T::TJ; j += T::kThreads) {
    if (j0 + j >= l.rows) break;
    int m = park[j].x;
#pragma unroll
    for (int i = 1; i < T::WI; ++i) m = max(m, park[i * T::TJ + j].x);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < T::WI; ++i) {
      const int2 v = park[i * T::TJ + j];
      if (v.x != -2147483647 - 1) sum += __int_as_float(v.y) * __builtin_amdgcn_exp2f(static_cast<float>(v.x - m) * k);
    }
    st.part[static_cast<long long>(j0 + j) * st.tiles + bi] = make_int2(m, __float_as_int(sum));
  }
}

template <class T>
__global__ __launch_bounds__(T::kThreads, T::kPerUnit) void vocab_grad_kernel(const VocabLogits l, const VocabGrad g) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int bi, bj;
  tile_of(blockIdx.x, (l.classes + T::TI - 1) / T::TI, (l.rows + T::TJ - 1) / T::TJ, &bi, &bj);
  const int i0 = bi * T::TI, j0 = bj * T::TJ;
  Product<T, false, false, v4i> p;
  p.run(l.w, l.a, i0, j0, 0, (l.features + kStageBytes - 1) / kStageBytes, l.w.row_bytes, l.a.row_bytes, smem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / T::WJ, wj = wave % T::WJ;
  const float k = exp2_scale(l);
  const int v0 = i0 + wi * T::BI * 16 + 4 * (lane >> 4);
  const int padded = (l.classes + 7) & ~7;
#pragma unroll
  for (int j = 0; j < T::BJ; ++j) {
    const int n = j0 + (wj * T::BJ + j) * 16 + (lane & 15);
    if (n >= l.rows) continue;
    const int32_t* const row = g.state + n * g.state_words;
    const int m = row[0];
    const float shift = static_cast<float>(kGradExponent) - __int_as_float(row[1]);
    const float coef = __int_as_float(row[2]);
    _Float16* const out = g.g + n * g.pitch;
#pragma unroll
    for (int i = 0; i < T::BI; ++i) {
      const int v = v0 + i * 16;
      if (v >= padded) continue;
      v4h o;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(fmaf(static_cast<float>(p.acc[i][j][r] - m), k, shift)) * coef;
        o[r] = static_cast<_Float16>(v + r < l.classes ? e : 0.0f);
      }
      *reinterpret_cast<v4h*>(out + v) = o;
    }
  }
}

__device__ inline uint16_t bf16_of(float f) {   // round to nearest, ties to even; NaN stays NaN
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40u);
  return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

__device__ inline int sums_exponent(const VocabSums& s) { return *s.exponent + s.bias + (s.exponent2 != nullptr ? *s.exponent2 : 0); }
__device__ inline float sums_weight(const VocabSums& s, int j) { return s.weight == nullptr ? s.t : s.t * s.weight[s.weight_n == 1 ? 0 : j]; }

template <class T, bool kYSlow>
__global__ __launch_bounds__(T::kThreads, T::kPerUnit) void vocab_sums_kernel(const VocabSums s) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int ti = (s.ni + T::TI - 1) / T::TI, tj = (s.nj + T::TJ - 1) / T::TJ;
  const int slice = blockIdx.x / (ti * tj);
  int bi, bj;
  tile_of(blockIdx.x - slice * ti * tj, ti, tj, &bi, &bj);
  const int i0 = bi * T::TI, j0 = bj * T::TJ;
  const int stages = (s.nk + 63) / 64;
  const int k0 = slice * s.steps;
  const int n = min(s.steps, stages - k0);
  const int end = min(s.nk, (k0 + n) * 64);      // steps
  Product<T, true, kYSlow, v4f> p;
  p.run(s.x, s.y, i0, j0, k0, n, end, kYSlow ? end : 2 * ((end + 7) & ~7), smem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / T::WJ, wj = wave % T::WJ;
  const int iw = i0 + wi * T::BI * 16 + 4 * (lane >> 4);
  const int e = sums_exponent(s);
#pragma unroll
  for (int j = 0; j < T::BJ; ++j) {
    const int jj = j0 + (wj * T::BJ + j) * 16 + (lane & 15);
    if (jj >= s.nj) continue;
    const float weight = s.part == nullptr ? sums_weight(s, jj) : 1.0f;
#pragma unroll
    for (int i = 0; i < T::BI; ++i) {
      const int ii = iw + i * 16;
      if (ii >= s.ni) continue;
      v4f v = p.acc[i][j];
      if (s.part != nullptr) {
        v4f* const at = reinterpret_cast<v4f*>(s.part + (static_cast<long long>(slice) * s.nj + jj) * s.part_pitch + ii);
        if (s.accumulate) v += *at;
        *at = v;
      } else {
        uint16_t* const at = s.out + static_cast<long long>(jj) * s.ni + ii;
        uint16_t b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) b[r] = bf16_of(ldexpf(v[r] * weight, e));
        if ((s.ni & 3) == 0) {
          *reinterpret_cast<uint64_t*>(at) = b[0] | static_cast<uint64_t>(b[1]) << 16 | static_cast<uint64_t>(b[2]) << 32 | static_cast<uint64_t>(b[3]) << 48;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (ii + r < s.ni) at[r] = b[r];
        }
      }
    }
  }
}

// adds the slices, scales, rounds; a lane takes four neighbours of a row
__global__ __launch_bounds__(256) void vocab_join_kernel(const VocabSums s) {
  const int quads = (s.ni + 3) / 4;
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= static_cast<long long>(quads) * s.nj) return;
  const int j = static_cast<int>(at / quads), i = static_cast<int>(at - static_cast<long long>(j) * quads) * 4;
  v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
  const float* p = s.part + j * s.part_pitch + i;
  const long long slice = static_cast<long long>(s.nj) * s.part_pitch;
  int k = 0;
  for (; k + 8 <= s.slices; k += 8) {
    v4f t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = *reinterpret_cast<const v4f*>(p + (k + u) * slice);
#pragma unroll
    for (int u = 0; u < 8; ++u) v += t[u];
  }
  for (; k < s.slices; ++k) v += *reinterpret_cast<const v4f*>(p + k * slice);
  const float weight = sums_weight(s, j);
  const int e = sums_exponent(s);
  uint16_t* const out = s.out + static_cast<long long>(j) * s.ni + i;
  for (int r = 0; r < 4 && i + r < s.ni; ++r) out[r] = bf16_of(ldexpf(v[r] * weight, e));
}

template <auto kernel>
int with_lds(int lds, const char* what) {   // more LDS than the default limit of a launch
  static bool done[kDeviceSlots];
  bool& set = done[device_slot()];
  if (set) return NITI_OK;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return fail(NITI_ERR_LAUNCH, "%s: %d bytes of LDS refused", what, lds);
  set = true;
  return NITI_OK;
}

template <class T>
int run_stats(const VocabLogits& l, const VocabStats& s, hipStream_t stream) {
  if (const int rc = with_lds<vocab_stats_kernel<T>>(T::kLds, "vocab_stats")) return rc;
  const long long tiles = static_cast<long long>((l.classes + T::TI - 1) / T::TI) * ((l.rows + T::TJ - 1) / T::TJ);
  hipLaunchKernelGGL(vocab_stats_kernel<T>, dim3(static_cast<unsigned>(tiles)), dim3(T::kThreads), T::kLds, stream, l, s);
  return check_launch("vocab_stats");
}
template <class T>
int run_grad(const VocabLogits& l, const VocabGrad& g, hipStream_t stream) {
  if (const int rc = with_lds<vocab_grad_kernel<T>>(T::kLds, "vocab_grad")) return rc;
  const long long tiles = static_cast<long long>((l.classes + T::TI - 1) / T::TI) * ((l.rows + T::TJ - 1) / T::TJ);
  hipLaunchKernelGGL(vocab_grad_kernel<T>, dim3(static_cast<unsigned>(tiles)), dim3(T::kThreads), T::kLds, stream, l, g);
  return check_launch("vocab_grad");
}
template <class T, bool kYSlow>
int run_sums(const VocabSums& s, hipStream_t stream) {
  if (const int rc = with_lds<vocab_sums_kernel<T, kYSlow>>(T::kLds, "vocab_sums")) return rc;
  const long long tiles = static_cast<long long>((s.ni + T::TI - 1) / T::TI) * ((s.nj + T::TJ - 1) / T::TJ) * s.slices;
  hipLaunchKernelGGL((vocab_sums_kernel<T, kYSlow>), dim3(static_cast<unsigned>(tiles)), dim3(T::kThreads), T::kLds, stream, s);
  return check_launch("vocab_sums");
}

long long tiles_of(long long ni, long long nj, int ti, int tj) { return ((ni + ti - 1) / ti) * ((nj + tj - 1) / tj); }
bool large_tiles(int ni, int nj) { return tiles_of(ni, nj, 256, 256) >= 200; }

}  // namespace

int launch_vocab_stats(const VocabLogits& l, const VocabStats& s, hipStream_t stream) {
  return l.rows <= 32 ? run_stats<TileFew>(l, s, stream) : run_stats<TileLarge>(l, s, stream);
}

int launch_vocab_grad(const VocabLogits& l, const VocabGrad& g, hipStream_t stream) {
  if (l.rows <= 32) return run_grad<TileFew>(l, g, stream);
  return large_tiles(l.classes, l.rows) ? run_grad<TileLarge>(l, g, stream) : run_grad<TileMiddle>(l, g, stream);
}

void vocab_sums_plan(int ni, int nj, int nk, int* slices, int* steps) {
  const long long tiles = nj <= 32 ? tiles_of(ni, nj, 256, 32) : (large_tiles(ni, nj) ? tiles_of(ni, nj, 256, 256) : tiles_of(ni, nj, 128, 128));
  const int stages = (nk + 63) / 64;
  long long want = tiles >= 200 ? 1 : (512 + tiles - 1) / tiles;
  if (want > stages / 4) want = stages / 4;
  if (want < 1) want = 1;
  *steps = static_cast<int>((stages + want - 1) / want);
  *slices = (stages + *steps - 1) / *steps;
}

int launch_vocab_sums(const VocabSums& s, bool y_slow, hipStream_t stream) {
  if (s.nj <= 32) return y_slow ? run_sums<TileFew, true>(s, stream) : run_sums<TileFew, false>(s, stream);
  if (large_tiles(s.ni, s.nj)) return y_slow ? run_sums<TileLarge, true>(s, stream) : run_sums<TileLarge, false>(s, stream);
  return y_slow ? run_sums<TileMiddle, true>(s, stream) : run_sums<TileMiddle, false>(s, stream);
}

int launch_vocab_join(const VocabSums& s, hipStream_t stream) {
  const long long quads = static_cast<long long>((s.ni + 3) / 4) * s.nj;
  hipLaunchKernelGGL(vocab_join_kernel, dim3(static_cast<unsigned>((quads + 255) / 256)), dim3(256), 0, stream, s);
  return check_launch("vocab_join");
}

}  // namespace niti
