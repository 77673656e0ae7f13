// Products of the losses over a large vocabulary (vocab.h): the logits' statistics, a piece of their gradient, and the sums of the
// two gradients behind it.  One tile product serves all three.
//
// Tile: TI x TJ results of sum_k x[i][k] y[j][k]; lane l of a wavefront holds for each 16 x 16 block column j = l % 16 and the rows
// i = 4 (l / 16) .. + 4 (v_mfma_i32_16x16x64_i8 or v_mfma_f32_16x16x32_f16).  A stage is 128 bytes of an int8 reduction, 64 steps of a
// 16-bit one, in a ring of buffers, filled by buffer_load ... lds while others are multiplied.  An operand lies in a stage
//   kFast    as whole 128-byte lines of its rows, 16-byte pieces XOR-swizzled by row / 2 so that the 16 rows a fragment read takes lie
//            in different banks
//   kSlow16  as stored with a slow reduction index, 64 steps of 16-bit columns, transposed by ds_read_b64_tr_b16, its 32-byte pieces
//            XOR-swizzled by the step
//   kSlow8   the same of int8 columns, transposed by ds_read_b64_tr_b8 and made 16-bit floats in registers (exact)
//
// What bounds the 256 x 256 tile is the clock that its power leaves: over 8192 x 8192 x 4096 the statistics, a piece of the gradient and the two
// sums took 264, 235, 430 and 390 us on data and 189, 180, 312 and 297 us, in the same code, on zeros, and by the counters as many clocks, of 1.83 GHz
// (gradient 2.00) and 2.3 (2.4).  In 65, 51 and 68 % of the clocks the matrix units are busy.  What was measured on the way there, as sums of one gradient and of the other: loads issued all at once behind the barrier 464 and 437, spread
// over the products of half a stage 427 and 393; with the loads left out 381 and 359, with products alone 335 and 308; two phases of half
// the rows with a barrier each 446 and 407; four wavefronts of 128 x 128, whose sums move between register files, 635 and 589.
#include "lds_asm.h"
#include "vocab.h"

namespace niti {
namespace {

constexpr int kFar = static_cast<int>(0x80000000u);   // beyond every buffer: reads as zero
constexpr int kStageBytes = 128;                      // of a fast reduction
constexpr int kNone = -2147483647 - 1;                // below every logit

enum Layout { kFast, kSlow16, kSlow8 };
constexpr int stage_bytes(int r, Layout l) { return l == kSlow8 ? 64 * r : kStageBytes * r; }

template <int TI_, int TJ_, int WI_, int WJ_, int RING_, int PER_UNIT, bool APART = false>
struct Tile {
  static constexpr int TI = TI_, TJ = TJ_, WI = WI_, WJ = WJ_, RING = RING_;     // RING: buffers
  static constexpr int kWaves = WI * WJ, kThreads = 64 * kWaves;
  static constexpr int BI = TI / WI / 16, BJ = TJ / WJ / 16;   // 16 x 16 blocks of a wavefront
  static constexpr bool kApart = APART;                        // see Apart
  static constexpr int kRings = kApart ? kWaves : 1;
  static constexpr int kLds = kRings * RING * (TI + TJ) * kStageBytes;
  static constexpr int kPerUnit = PER_UNIT;      // workgroups per unit that the registers are cut for
  static constexpr bool kInTurn = TI == 256;     // logits: a workgroup takes several tiles in turn, with LDS for their ends behind the ring
  static constexpr int kLdsLogits = kLds + (kInTurn ? 2 * TI * 16 * WJ : 0);
};
typedef Tile<256, 256, 2, 4, 2, 1> TileLarge;
typedef Tile<128, 128, 2, 2, 2, 2> TileMiddle;
typedef Tile<64, 64, 2, 2, 2, 4> TileSmall;
typedef Tile<64, 64, 2, 2, 4, 2> TileDeep;      // few tiles: what counts is how soon the loads are out
typedef Tile<128, 32, 4, 1, 4, 2> TileFew;
typedef Tile<128, 32, 4, 1, 3, 4> TileFewSums;
typedef Tile<64, 32, 4, 1, 3, 2, true> TileFewApart;      // few tiles of long reductions: a stage of the reduction for each wavefront
typedef Tile<64, 64, 2, 2, 2, 2, true> TileSmallApart;
typedef Tile<128, 128, 2, 2, 1, 4> TileShort;   // short reductions: nothing overlaps within a tile, but with three other tiles of a unit

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

// eight int8 values as 16-bit floats, exactly: a byte b + 128 under the exponent of 1024 is 1024 + 128 + b
__device__ inline v4i widen8(v2i b) {
  const v2h bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  v4i o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned u = static_cast<unsigned>(b[h]) ^ 0x80808080u;
    const unsigned lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    o[2 * h] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, lo) + bias);
    o[2 * h + 1] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, hi) + bias);
  }
  return o;
}

// One operand's way from memory to its stages: R rows (or columns, where the reduction index is slow).
template <int R, Layout L, int kWaves>
struct Source {
  static constexpr bool kSlow = L != kFast;
  static constexpr int kStage = stage_bytes(R, L);
  static constexpr int kInstructions = kStage / 1024;                       // of a stage
  static constexpr int kLoads = kInstructions / kWaves;                     // of a wavefront, 16 bytes per lane each
  static constexpr int kRowBytes = L == kFast ? kStageBytes : (L == kSlow16 ? 2 * R : R);
  static constexpr int kRowsPerLoad = 1024 / kRowBytes;
  static constexpr int kPieces = kRowBytes / 16;
  static_assert(kInstructions % kWaves == 0, "the same number of each wavefront");

  const char* base;
  long long left;        // bytes from base to the end of the matrix
  long long advance;     // per stage
  int fast_left;         // bytes of the reduction left in a row (kFast)
  int voff[kLoads];
  int piece;

  // what a step's pieces are swizzled by: the steps that 32 lanes read at once differ in it (kSlow16: four of each 16-lane group, groups
  // eight steps apart; kSlow8: eight of each)
  static __device__ int turn(int k) { return (L == kSlow16 ? (k & 3) | (((k >> 3) & 1) << 2) : k & 15) & (R / 16 - 1); }

  __device__ void lanes(const VocabOperand& o) {
    const int lane = threadIdx.x & 63;
    const int wave = kWaves == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    piece = 0;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int row = (q * kWaves + wave) * kRowsPerLoad + lane / kPieces;
      const int slot = lane % kPieces;
      const int c = L == kFast ? slot ^ ((row >> 1) & 7) : (L == kSlow16 ? slot ^ (2 * turn(row)) : slot ^ turn(row));
      if (!kSlow && q == 0) piece = c * 16;
      voff[q] = static_cast<int>(row * o.pitch) + c * 16;
    }
  }
  // first: first row (fast) or column (slow) of the tile; k0: first stage; k_end: end of the reduction's range in bytes (fast) or steps (slow)
  __device__ void seek(const VocabOperand& o, int first, int k0, int k_end) {
    const char* const p = static_cast<const char*>(o.p);
    if (kSlow) {
      const long long skip = static_cast<long long>(k0) * 64 * o.pitch + (L == kSlow16 ? 2LL : 1LL) * first;
      base = p + skip;
      left = (k_end - 1) * o.pitch + o.row_bytes - skip;
      advance = 64 * o.pitch;
      fast_left = 0;
    } else {
      const long long skip = first * o.pitch + static_cast<long long>(k0) * kStageBytes;
      base = p + skip;
      left = (o.rows - 1) * o.pitch + o.row_bytes - skip;
      advance = kStageBytes;
      fast_left = k_end - k0 * kStageBytes;
    }
  }

  // the stage that load() fetches instructions of; next() moves on
  __device__ __amdgpu_buffer_rsrc_t stage() const {
    const int n = left <= 0 ? 0 : (left > 0x7fffffffLL ? 0x7fffffff : static_cast<int>(left));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, n, 0x00020000);
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned lds, int q) const {
    const int wave = kWaves == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int turned = (q * kWaves * kRowsPerLoad / 2 & 7) << 4;      // rows of this load have their pieces turned by this against load 0's
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, NITI_LDS_AT(lds + (q * kWaves + wave) * 1024), 16, kSlow || (piece ^ turned) < fast_left ? voff[q] : kFar, 0, 0, 0);
  }
  template <int BY = 1>
  __device__ void next() {
    base += BY * advance;
    left -= BY * advance;
    fast_left -= BY * kStageBytes;
  }
};

// Fragments of B blocks of 16 rows / columns, starting at block `first` of the operand's stages at LDS address `lds`.
template <int R, int B, Layout L>
struct Fragments {
  static constexpr int kAddr = L == kFast ? 2 : B;
  unsigned addr[kAddr];
  // halves of a stage, of up to two stages (those that a tile does not use are no registers)
  v2i lo[4][L == kFast ? 1 : B], hi[4][L == kSlow16 ? B : 1];
  v4i whole[4][L == kFast ? B : 1];

  __device__ void init(unsigned lds, int first) {
    const int lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    if constexpr (L == kFast) {
      addr[0] = lds + (first * 16 + i) * kStageBytes + ((g ^ (i >> 1)) << 4);
      addr[1] = addr[0] ^ 64;
    } else {
      const int step = 8 * g + (L == kSlow16 ? i >> 2 : i >> 1);
      const int t = Source<R, L, 1>::turn(step);     // the same for the other steps that this lane names
#pragma unroll
      for (int b = 0; b < B; ++b)
        addr[b] = L == kSlow16 ? lds + step * (2 * R) + (((first + b) ^ t) << 5) + (i & 3) * 8 : lds + step * R + (((first + b) ^ t) << 4) + (i & 1) * 8;
    }
  }
  __device__ void other_buffer(int step) {
#pragma unroll
    for (int b = 0; b < kAddr; ++b) addr[b] += step;
  }
  // block BLK of half H % 2 into register set H
  template <int H, int BLK>
  __device__ void read() {
    constexpr int SUB = H & 1;
    if constexpr (L == kSlow16) {
      lo[H][BLK] = lds_read_tr16<SUB * 64 * R>(addr[BLK]);
      hi[H][BLK] = lds_read_tr16<SUB * 64 * R + 8 * R>(addr[BLK]);
    } else if constexpr (L == kSlow8) {
      lo[H][BLK] = lds_read_tr8<SUB * 32 * R>(addr[BLK]);
    } else {
      whole[H][BLK] = lds_read_b128_at<BLK * 16 * kStageBytes>(addr[SUB]);
    }
  }
  // behind a settle: the reads of set H are in their registers
  template <int H>
  __device__ void landed() {
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if constexpr (L == kSlow16) asm volatile("" : "+v"(lo[H][b]), "+v"(hi[H][b]));
      else if constexpr (L == kSlow8) asm volatile("" : "+v"(lo[H][b]));
      else asm volatile("" : "+v"(whole[H][b]));
    }
  }
  template <int H, int BLK>
  __device__ v4i get() const {
    if constexpr (L == kSlow16) return v4i{lo[H][BLK][0], lo[H][BLK][1], hi[H][BLK][0], hi[H][BLK][1]};
    else if constexpr (L == kSlow8) return widen8(lo[H][BLK]);
    else return whole[H][BLK];
  }
};

__device__ inline v4i multiply(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
__device__ inline v4f multiply(v4i a, v4i b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Main loop.  Half a stage's fragments are read while the other half is multiplied, and the barrier lies between the halves: behind it
// the next stage's first half is requested along with the second half's products, and the loads of the stage after that go out, so no
// product waits for the reads behind a barrier.  The fragments carried into the next turn have landed by the end of one.
template <class T, Layout LX, Layout LY, class Acc>
struct Product {
  Source<T::TI, LX, T::kWaves> sx;
  Source<T::TJ, LY, T::kWaves> sy;
  Fragments<T::TI, T::BI, LX> fx;
  Fragments<T::TJ, T::BJ, LY> fy;
  Acc acc[T::BI][T::BJ];
  unsigned ldsx, ldsy;
  static constexpr int kStageX = stage_bytes(T::TI, LX), kStageY = stage_bytes(T::TJ, LY);
  static constexpr int kLoadsX = Source<T::TI, LX, T::kWaves>::kLoads, kLoadsY = Source<T::TJ, LY, T::kWaves>::kLoads;
  static_assert(T::RING * (kStageX + kStageY) <= T::kLds, "stages fit");

  // instruction q of a stage's loads into buffer buf
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rx, __amdgpu_buffer_rsrc_t ry, int buf, int q) const {
    if (q < kLoadsX) sx.load(rx, ldsx + buf * kStageX, q);
    else sy.load(ry, ldsy + buf * kStageY, q - kLoadsX);
  }
  __device__ void issue(int buf) {
    const __amdgpu_buffer_rsrc_t rx = sx.stage(), ry = sy.stage();
    static_for<kLoadsX + kLoadsY>([&](auto q) { load(rx, ry, buf, decltype(q)::value); });
    sx.next();
    sy.next();
  }
  // Products of half SUB; half NEXT is read in between, and where kLoad the next stage that has no buffer yet goes out into buffer buf, spread over the
  // products: a unit's loads pass at 64 bytes a clock, and a wavefront waits at a load that finds the queue full
  template <int SUB, int NEXT, bool kLoad>
  __device__ void half(int buf) {
    const __amdgpu_buffer_rsrc_t rx = sx.stage(), ry = sy.stage();
    static_for<(T::BJ > T::BI ? T::BJ - T::BI : 0)>([&](auto j) { fy.template read<NEXT, T::BI + decltype(j)::value>(); });
    static_for<T::BI>([&](auto i) {
      constexpr int I = decltype(i)::value;
      if constexpr (I < T::BJ) fy.template read<NEXT, I>();
      fx.template read<NEXT, I>();
      __builtin_amdgcn_s_setprio(1);
      const v4i x = fx.template get<SUB, I>();
      static_for<T::BJ>([&](auto j) {
        constexpr int J = decltype(j)::value;
        acc[I][J] = multiply(x, fy.template get<SUB, J>(), acc[I][J]);
      });
      __builtin_amdgcn_s_setprio(0);
      if constexpr (kLoad) {
        constexpr int kAll = kLoadsX + kLoadsY, kFrom = I * kAll / T::BI, kTo = (I + 1) * kAll / T::BI;
        static_for<kTo - kFrom>([&](auto q) { load(rx, ry, buf, kFrom + decltype(q)::value); });
      }
      __builtin_amdgcn_sched_barrier(0);      // reads, products and loads stay in this order
    });
    if constexpr (kLoad) {
      sx.next();
      sy.next();
    }
    lds_settle<0>();
    fx.template landed<NEXT>();
    fy.template landed<NEXT>();
  }

  // all reads / products of register set H
  template <int H>
  __device__ void read_all() {
    static_for<T::BJ>([&](auto j) { fy.template read<H, decltype(j)::value>(); });
    static_for<T::BI>([&](auto i) { fx.template read<H, decltype(i)::value>(); });
  }
  template <int H>
  __device__ void landed() {
    fx.template landed<H>();
    fy.template landed<H>();
  }
  template <int H>
  __device__ void multiply_all() {
    static_for<T::BI>([&](auto i) {
      constexpr int I = decltype(i)::value;
      const v4i x = fx.template get<H, I>();
      static_for<T::BJ>([&](auto j) { acc[I][decltype(j)::value] = multiply(x, fy.template get<H, decltype(j)::value>(), acc[I][decltype(j)::value]); });
    });
  }
  // at most N of a wavefront's loads are still under way, for all wavefronts
  template <int N>
  __device__ void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  // A whole stage of a small tile, whose fragments are in sets 2 A and 2 A + 1: a half's few products would not cover the way of the other
  // half's fragments, so those of the next stage are all requested ahead of this one's products.
  template <int A>
  __device__ void whole_stage(int& buf) {
    constexpr int B = 1 - A;
    stage_barrier<(T::RING - 2) * (kLoadsX + kLoadsY)>();      // the next stage has landed; this one's fragments are with every wavefront
    const int step = buf + 1 < T::RING ? 1 : 1 - T::RING;
    fx.other_buffer(step * kStageX);
    fy.other_buffer(step * kStageY);
    read_all<2 * B>();
    read_all<2 * B + 1>();
    issue(buf);
    buf += step;
    multiply_all<2 * A>();
    multiply_all<2 * A + 1>();
    lds_settle<0>();
    landed<2 * B>();
    landed<2 * B + 1>();
  }

  __device__ void lanes(const VocabOperand& x, const VocabOperand& y, char* smem) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ldsx = lds_addr(smem);
    ldsy = ldsx + T::RING * kStageX;
    sx.lanes(x);
    sy.lanes(y);
    fx.init(ldsx, (wave / T::WJ) * T::BI);
    fy.init(ldsy, (wave % T::WJ) * T::BJ);
  }
  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int j = 0; j < T::BJ; ++j) acc[i][j] = Acc{0, 0, 0, 0};
  }

  // x, y: operands; i0, j0: the tile's corner; range of the reduction: stages k0 .. k0 + n, ending at x_end and y_end (bytes or steps)
  __device__ void run(const VocabOperand& x, const VocabOperand& y, int i0, int j0, int k0, int n, int x_end, int y_end, char* smem) {
    lanes(x, y, smem);
    sx.seek(x, i0, k0, x_end);
    sy.seek(y, j0, k0, y_end);
    clear();
    if constexpr (T::RING == 1) {      // a stage after the other, half after half
      for (int s = 0; s < n; ++s) {
        issue(0);
        tile_sync();
        static_for<2>([&](auto h) {
          constexpr int H = decltype(h)::value;
          read_all<H>();
          lds_settle<0>();
          landed<H>();
          multiply_all<H>();
          __builtin_amdgcn_sched_barrier(0);
        });
        tile_sync();
      }
      return;
    }
    // loads of the stages behind the last are issued like the others: they are out of range, and what they clear is not multiplied
    static_for<T::RING>([&](auto b) { issue(decltype(b)::value); });
    constexpr int kStageLoads = kLoadsX + kLoadsY;       // of a wavefront
    stage_barrier<(T::RING - 1) * kStageLoads>();
    read_all<0>();
    if constexpr (T::BI * T::BJ <= 4) read_all<1>();
    lds_settle<0>();
    landed<0>();
    int buf = 0;
    if constexpr (T::BI * T::BJ <= 4) {
      landed<1>();
      for (int s = 0; s < n; s += 2) {
        whole_stage<0>(buf);
        if (s + 1 < n) whole_stage<1>(buf);
      }
    } else {
      for (int s = 0; s < n; ++s) {
        half<0, 1, false>(buf);
        stage_barrier<(T::RING - 2) * kStageLoads>();      // the next stage has landed, and this one's buffer has been read by every wavefront
        const int step = buf + 1 < T::RING ? 1 : 1 - T::RING;
        fx.other_buffer(step * kStageX);
        fy.other_buffer(step * kStageY);
        half<1, 0, true>(buf);
        buf += step;
      }
    }
    tile_sync();            // the buffers are free
  }
};

// The same sums where a launch is few tiles: what counts is a tile's walk along its reduction, 0.3 - 0.4 us a stage where wavefronts take
// stages together (barrier, fragments and products one after the other; a ring of eight is no faster).  Each takes every kWaves-th stage
// here, for the whole tile, in a ring of its own and without barriers; their sums meet in LDS at the end, in the order of the wavefronts, and
// go back to the registers as Product leaves them.  Sums of a tile of 16 x 512 over 1000 classes, 16 stages, 6.7 us together.
template <class T, Layout LX, Layout LY, class Acc>
struct Apart {
  static constexpr int PI = T::TI / 16, PJ = T::TJ / 16;
  Source<T::TI, LX, 1> sx;
  Source<T::TJ, LY, 1> sy;
  Fragments<T::TI, PI, LX> fx;
  Fragments<T::TJ, PJ, LY> fy;
  Acc acc[T::BI][T::BJ];
  static constexpr int kStageX = stage_bytes(T::TI, LX), kStageY = stage_bytes(T::TJ, LY);
  static constexpr int kStageLoads = Source<T::TI, LX, 1>::kLoads + Source<T::TJ, LY, 1>::kLoads;
  static_assert(T::RING == 2 || T::RING == 3, "the waits");
  static_assert(T::kWaves * PI * PJ * 1024 <= T::kWaves * T::RING * (kStageX + kStageY), "the sums meet where the rings were");

  __device__ void issue(unsigned ldsx, unsigned ldsy, int buf) {
    const __amdgpu_buffer_rsrc_t rx = sx.stage(), ry = sy.stage();
    static_for<Source<T::TI, LX, 1>::kLoads>([&](auto q) { sx.load(rx, ldsx + buf * kStageX, decltype(q)::value); });
    static_for<Source<T::TJ, LY, 1>::kLoads>([&](auto q) { sy.load(ry, ldsy + buf * kStageY, decltype(q)::value); });
    sx.template next<T::kWaves>();
    sy.template next<T::kWaves>();
  }
  __device__ void run(const VocabOperand& x, const VocabOperand& y, int i0, int j0, int k0, int n, int x_end, int y_end, char* smem) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned ldsx = lds_addr(smem) + wave * T::RING * (kStageX + kStageY), ldsy = ldsx + T::RING * kStageX;
    sx.lanes(x);
    sy.lanes(y);
    fx.init(ldsx, 0);
    fy.init(ldsy, 0);
    sx.seek(x, i0, k0 + wave, x_end);
    sy.seek(y, j0, k0 + wave, y_end);
    Acc own[PI][PJ];
#pragma unroll
    for (int i = 0; i < PI; ++i)
#pragma unroll
      for (int j = 0; j < PJ; ++j) own[i][j] = Acc{0, 0, 0, 0};
    const int rounds = (n - wave + T::kWaves - 1) / T::kWaves;      // stages of this wavefront
    static_for<T::RING>([&](auto b) {
      if (decltype(b)::value < rounds) issue(ldsx, ldsy, decltype(b)::value);
    });
    int buf = 0;
    for (int left = rounds - 1; left >= 0; --left) {      // stages behind this one, of which RING - 1 are under way
      if (left >= T::RING - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::RING - 1) * kStageLoads) : "memory");
      else if (left == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kStageLoads) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      static_for<2>([&](auto h) {
        constexpr int H = decltype(h)::value;
        static_for<PJ>([&](auto j) { fy.template read<H, decltype(j)::value>(); });
        static_for<PI>([&](auto i) { fx.template read<H, decltype(i)::value>(); });
      });
      lds_settle<0>();
      fx.template landed<0>();
      fx.template landed<1>();
      fy.template landed<0>();
      fy.template landed<1>();
      if (left >= T::RING) issue(ldsx, ldsy, buf);
      static_for<2>([&](auto h) {
        constexpr int H = decltype(h)::value;
        static_for<PI>([&](auto i) {
          constexpr int I = decltype(i)::value;
          const v4i xi = fx.template get<H, I>();
          static_for<PJ>([&](auto j) { own[I][decltype(j)::value] = multiply(xi, fy.template get<H, decltype(j)::value>(), own[I][decltype(j)::value]); });
        });
      });
      const int step = buf + 1 < T::RING ? 1 : 1 - T::RING;
      fx.other_buffer(step * kStageX);
      fy.other_buffer(step * kStageY);
      buf += step;
    }
    tile_sync();
    Acc* const meet = reinterpret_cast<Acc*>(smem) + lane;
#pragma unroll
    for (int i = 0; i < PI; ++i)
#pragma unroll
      for (int j = 0; j < PJ; ++j) meet[((wave * PI + i) * PJ + j) * 64] = own[i][j];
    __syncthreads();
    const int wi = wave / T::WJ, wj = wave % T::WJ;
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int j = 0; j < T::BJ; ++j) {
        const int at = (wi * T::BI + i) * PJ + wj * T::BJ + j;
        acc[i][j] = meet[at * 64];
#pragma unroll
        for (int w = 1; w < T::kWaves; ++w) acc[i][j] += meet[(w * PI * PJ + at) * 64];
      }
    __syncthreads();
  }
};
template <class T, Layout LX, Layout LY, class Acc>
using Sums = std::conditional_t<T::kApart, Apart<T, LX, LY, Acc>, Product<T, LX, LY, Acc>>;

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

// Logits of the tiles first, first + step, ... of `total` in turn: the last stages of a tile already load the first ones of the next, so
// between two tiles there is only what `done` does with the first one's sums.  done(sums, i0, j0) waits for the loads under way
// (s_waitcnt vmcnt(0)) in front of its first store - the next barrier then need not wait for its stores - and ends with a barrier if it uses LDS,
// which is its own behind the ring.
template <class T, class F>
__device__ inline void logit_tiles(const VocabLogits& l, int first, int step, int total, int ti, int tj, char* smem, F done) {
  Product<T, kFast, kFast, v4i> p;
  static_assert(T::RING == 2 && T::BI * T::BJ > 4, "the two loads ahead of the loop; the loop of half stages");
  const int n = (l.features + kStageBytes - 1) / kStageBytes;
  int load_tile = first, load_stage = 0;
  const auto seek = [&] {
    int bi = 0, bj = 0;
    if (load_tile < total) tile_of(load_tile, ti, tj, &bi, &bj);
    p.sx.seek(l.w, bi * T::TI, 0, l.w.row_bytes);
    p.sy.seek(l.a, bj * T::TJ, 0, l.a.row_bytes);
    if (load_tile >= total) p.sx.left = p.sy.left = 0;      // nothing behind the last tile
  };
  const auto loaded = [&] {
    if (++load_stage == n) {
      load_stage = 0;
      load_tile += step;
      seek();
    }
  };
  p.lanes(l.w, l.a, smem);
  seek();
  p.issue(0);
  loaded();
  p.issue(1);
  loaded();
  p.template stage_barrier<Product<T, kFast, kFast, v4i>::kLoadsX + Product<T, kFast, kFast, v4i>::kLoadsY>();
  int buf = 0;
  for (int tile = first; tile < total; tile += step) {
    p.clear();
    p.template read_all<0>();
    lds_settle<0>();
    p.template landed<0>();
    for (int s = 0; s < n; ++s) {
      p.template half<0, 1, false>(buf);
      if (s == 0 && tile != first) {      // everything but the last tile's stores has been waited for
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      } else {
        p.template stage_barrier<0>();
      }
      const int turn = buf == 0 ? 1 : -1;
      p.fx.other_buffer(turn * p.kStageX);
      p.fy.other_buffer(turn * p.kStageY);
      p.template half<1, 0, true>(buf);
      loaded();
      buf ^= 1;
    }
    int bi, bj;
    tile_of(tile, ti, tj, &bi, &bj);
    done(p.acc, bi * T::TI, bj * T::TJ, bi);
  }
  tile_sync();
}

// k of vocab.h, finite: an overflow would make 0 k a NaN where it stands for a difference of nothing
__device__ inline float exp2_scale(const VocabLogits& l) {
  const float k = ldexpf(1.44269504088896340736f * l.inv_t, *l.exp_a + *l.exp_w);
  return fminf(k, 3.402823466e38f);
}

// folds the values of the lanes i, i ^ 16, i ^ 32, i ^ 48, which hold one column's rows
template <class F>
__device__ inline int fold_quarters(int v, F f) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = f(static_cast<int>(a[0]), static_cast<int>(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return f(static_cast<int>(b[0]), static_cast<int>(b[1]));
}

// sixteen bytes of a row of which `left` are left (a multiple of four; what lies behind the row is not touched)
__device__ inline v4i row_piece(const char* p, int left) {
  if (left >= 16) return *reinterpret_cast<const v4i*>(p);
  const int* const w = reinterpret_cast<const int*>(p);
  return v4i{left > 0 ? w[0] : 0, left > 4 ? w[1] : 0, left > 8 ? w[2] : 0, 0};
}

constexpr int kPlaces = 8;     // of a row, whose products a wavefront makes at a time

// Logits of the targets: a wavefront takes eight places of a row, its lanes sixteen features each, the loads of all in flight together.
// Bound by the gathered rows' way: 64 places of 8192 rows of 2048 features 139 us, 1.07 GB at 7.7 TB/s, most of it out of the caches.
__device__ inline void dots_block(const VocabLogits& l, const VocabTargets& t, int block, int waves) {
  const int lane = threadIdx.x & 63;
  const int groups = (t.top + kPlaces - 1) / kPlaces;
  const long long unit = static_cast<long long>(block) * waves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long row = unit / groups;
  if (row >= l.rows) return;
  const int j0 = static_cast<int>(unit - row * groups) * kPlaces;
  const v4i* const arow = reinterpret_cast<const v4i*>(static_cast<const char*>(l.a.p) + row * l.a.pitch);
  const int pieces = l.a.row_bytes / 16;
  // a lane per place asks for its class
  const int mine = lane < kPlaces && j0 + lane < t.top ? vocab_target(t, row * t.top + j0 + lane, l.classes) : -1;
  v4i x = lane < pieces ? arow[lane] : v4i{0, 0, 0, 0};
  const char* w[kPlaces];
  int s[kPlaces];
#pragma unroll
  for (int u = 0; u < kPlaces; ++u) {
    const int c = __builtin_amdgcn_readlane(mine, u);
    w[u] = c < 0 ? nullptr : static_cast<const char*>(l.w.p) + c * l.w.pitch;
    s[u] = 0;
  }
  for (int p = lane; p < pieces; p += 64) {
    if (p >= 64) x = arow[p];
    v4i y[kPlaces];
#pragma unroll
    for (int u = 0; u < kPlaces; ++u) y[u] = w[u] != nullptr ? row_piece(w[u] + 16 * p, l.w.row_bytes - 16 * p) : v4i{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < kPlaces; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u] = __builtin_amdgcn_sdot4(x[i], y[u][i], s[u], false);
  }
  int out = 0;
#pragma unroll
  for (int u = 0; u < kPlaces; ++u)
    if (w[u] != nullptr) {
      const int all = wave_add(s[u]);
      out = lane == u ? all : out;
    }
  if (lane < kPlaces && j0 + lane < t.top) t.state[row * vocab_state_words(t.top) + 4 + 2 * (j0 + lane)] = out;
}

__global__ __launch_bounds__(256) void vocab_dots_kernel(const VocabLogits l, const VocabTargets t) { dots_block(l, t, blockIdx.x, 4); }

// The thread's index, anew: what is computed from it is not kept in registers through the main loop in front.
__device__ inline int thread_anew() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// Statistics of a tile's sums.  `park`: [WI][TJ] pairs
template <class T>
__device__ inline void stats_of(const VocabLogits& l, const VocabStats& st, const v4i (&acc)[T::BI][T::BJ], float k, int i0, int j0, int bi, int2* park) {
  const int thread = thread_anew(), lane = thread & 63;
  const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  const int wi = wave / T::WJ, wj = wave % T::WJ;
  const int v0 = i0 + wi * T::BI * 16 + 4 * (lane >> 4);
  const bool whole = i0 + T::TI <= l.classes;
#pragma unroll
  for (int j = 0; j < T::BJ; ++j) {
    int m = kNone;
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (whole || v0 + i * 16 + r < l.classes) m = max(m, acc[i][j][r]);
    m = fold_quarters(m, [](int a, int b) { return max(a, b); });
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (whole || v0 + i * 16 + r < l.classes) sum += __builtin_amdgcn_exp2f(static_cast<float>(acc[i][j][r] - m) * k);
    sum = __int_as_float(fold_quarters(__float_as_int(sum), [](int a, int b) { return __float_as_int(__int_as_float(a) + __int_as_float(b)); }));
    if (lane < 16) park[wi * T::TJ + (wj * T::BJ + j) * 16 + lane] = make_int2(m, __float_as_int(sum));
  }
  tile_sync();
  for (int j = thread; j < T::TJ; j += T::kThreads) {
    if (j0 + j >= l.rows) break;
    int m = park[j].x;
#pragma unroll
    for (int i = 1; i < T::WI; ++i) m = max(m, park[i * T::TJ + j].x);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < T::WI; ++i) {
      const int2 v = park[i * T::TJ + j];
      if (v.x != kNone) sum += __int_as_float(v.y) * __builtin_amdgcn_exp2f(static_cast<float>(v.x - m) * k);
    }
    st.part[static_cast<long long>(j0 + j) * st.tiles + bi] = make_int2(m, __float_as_int(sum));
  }
}

// Bound by the products: 8192 rows of 4096 features over 131072 classes 3.14 - 3.37 ms on three cards, 2.6 - 2.8 POP/s; few rows by the weights' way: 16 rows over
// 32000 classes of 4096 21 us, 131 MB at 6.2 TB/s called again and again, partly out of the last-level cache.  A pair per row and tile of
// classes is all that leaves.
// Statistics of the tiles, or - the first `others` workgroups, a multiple of eight - the targets' logits, which depend on nothing else
// either.  Large tiles: each workgroup takes several in turn.
template <class T>
__global__ __launch_bounds__(T::kThreads, T::kPerUnit) void vocab_stats_kernel(const VocabLogits l, const VocabStats st, const VocabTargets targets, int others) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  if (static_cast<int>(blockIdx.x) < others) {
    dots_block(l, targets, blockIdx.x, T::kWaves);
    return;
  }
  const int ti = (l.classes + T::TI - 1) / T::TI, tj = (l.rows + T::TJ - 1) / T::TJ;
  const int block = blockIdx.x - others;
  const float k = exp2_scale(l);
  if constexpr (T::kInTurn) {
    int2* const park = reinterpret_cast<int2*>(smem + T::kLds);
    logit_tiles<T>(l, block, gridDim.x - others, ti * tj, ti, tj, smem, [&](const v4i(&acc)[T::BI][T::BJ], int i0, int j0, int bi) {
      stats_of<T>(l, st, acc, k, i0, j0, bi, park);
      __syncthreads();
    });
  } else {
    int bi, bj;
    tile_of(block, ti, tj, &bi, &bj);
    Sums<T, kFast, kFast, v4i> p;
    p.run(l.w, l.a, bi * T::TI, bj * T::TJ, 0, (l.features + kStageBytes - 1) / kStageBytes, l.w.row_bytes, l.a.row_bytes, smem);
    stats_of<T>(l, st, p.acc, k, bi * T::TI, bj * T::TJ, bi, reinterpret_cast<int2*>(smem));
  }
}

__device__ inline void widen_block(const VocabWiden& w, int block, int threads, char* smem) {
  float scale = 1.0f;
  int e = 0;
  if (w.weight != nullptr) {
    float* const most = reinterpret_cast<float*>(smem);
    float m = 0.0f;
    constexpr int kAhead = 8;       // loads under way together
    for (int i = threadIdx.x; i < w.rows; i += kAhead * threads) {
      float v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) v[u] = i + u * threads < w.rows ? w.weight[i + u * threads] : 0.0f;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) m = fmaxf(m, fabsf(v[u]));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int i = 0; i < threads / 64; ++i) m = fmaxf(m, most[i]);
    if (m > 0.0f) frexpf(fminf(m, 3.402823466e38f), &e);
    if (block == 0 && threadIdx.x == 0) *w.exponent = e;
  }
  const int pieces = (w.values + 15) / 16;
  const long long all = static_cast<long long>(w.rows) * pieces;
  for (long long at = static_cast<long long>(block) * threads + threadIdx.x; at < all; at += static_cast<long long>(w.blocks) * threads) {
    const long long row = all < 0x7fffffffLL ? static_cast<unsigned>(at) / static_cast<unsigned>(pieces) : at / pieces;
    const int c = static_cast<int>(at - row * pieces) * 16;
    union {
      int8_t b[16];
      v4i v;
    } u;
    u.v = row_piece(reinterpret_cast<const char*>(w.src + row * w.src_pitch + c), w.src_bytes - c);
    if (w.weight != nullptr) scale = ldexpf(w.weight[row], kRowExponent - e);
    v8h o[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i >> 3][i & 7] = static_cast<_Float16>(static_cast<float>(u.b[i]) * scale);
    v8h* const out = reinterpret_cast<v8h*>(w.dst + row * w.pitch + c);
    out[0] = o[0];
    out[1] = o[1];
  }
}

// A tile of 16-bit values on its way out: [TJ][TI], 16-byte pieces XOR-swizzled by the row, so that lanes that hold four neighbours of
// 16 different rows write to different banks and rows leave as whole lines.
template <class T>
struct Outgoing {
  static constexpr int kPieces = T::TI / 8;
  char* smem;
  __device__ char* at(int j, int piece) const { return smem + j * (2 * T::TI) + ((piece ^ (j & (kPieces - 1))) << 4); }
  __device__ void put(int j, int i, uint64_t four) const { *reinterpret_cast<uint64_t*>(at(j, i >> 3) + ((i & 4) << 1)) = four; }
  __device__ uint16_t* one(int j, int i) const { return reinterpret_cast<uint16_t*>(at(j, i >> 3)) + (i & 7); }
};

// sum_j q_j p 2^kGradExponent of four neighbouring classes of a row
__device__ inline uint64_t grad_of(v4i s, v4i row, float k, int v, int classes) {
  const float shift = static_cast<float>(kGradExponent) - __int_as_float(row[1]);
  const float coef = __int_as_float(row[2]);
  v4h o;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float e = __builtin_amdgcn_exp2f(fmaf(static_cast<float>(s[r] - row[0]), k, shift)) * coef;
    o[r] = static_cast<_Float16>(v + r < classes ? e : 0.0f);
  }
  return __builtin_bit_cast(uint64_t, o);
}
__device__ inline uint16_t target_grad(int bits) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(ldexpf(__int_as_float(bits), kGradExponent))); }

// A piece of the gradient.  Bound as the statistics: 8192 rows of 4096 features, 8192 classes 241 - 249 us (2.2 - 2.3 POP/s), 134 MB out among it;
// few rows by one workgroup's walk from its start to the last store.
template <class T>
__global__ __launch_bounds__(T::kThreads, T::kPerUnit) void vocab_grad_kernel(const VocabLogits l, const VocabGrad g) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  // the copies' workgroups (a multiple of eight) come first where the tiles' stay to the end, behind the tiles otherwise
  const int ti = (l.classes + T::TI - 1) / T::TI, tj = (l.rows + T::TJ - 1) / T::TJ;
  const int others = (g.widen_a.blocks + g.widen_w.blocks + 7) / 8 * 8;
  const int copy = T::kInTurn ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) - ti * tj;
  if (T::kInTurn ? copy < others : copy >= 0) {
    if (copy < g.widen_a.blocks) widen_block(g.widen_a, copy, T::kThreads, smem);
    else if (copy - g.widen_a.blocks < g.widen_w.blocks) widen_block(g.widen_w, copy - g.widen_a.blocks, T::kThreads, smem);
    return;
  }
  const float k = exp2_scale(l);
  const int padded = (l.classes + 7) & ~7;
  if constexpr (T::kInTurn) {
    // on its way out the tile passes in T::BJ parts of 16 rows per wavefront column through LDS of its own
    const Outgoing<T> out{smem + T::kLds};
    constexpr int kRows = 16 * T::WJ;
    const auto row_of = [](int r, int part) { return (r >> 4) * (16 * T::BJ) + part * 16 + (r & 15); };
    logit_tiles<T>(l, blockIdx.x - others, gridDim.x - others, ti * tj, ti, tj, smem, [&](const v4i(&acc)[T::BI][T::BJ], int i0, int j0, int) {
      const int thread = thread_anew(), lane = thread & 63;
      const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
      const int wi = wave / T::WJ, wj = wave % T::WJ;
      v4i rows[T::BJ];
#pragma unroll
      for (int part = 0; part < T::BJ; ++part) {
        const int n = j0 + row_of(wj * 16 + (lane & 15), part);
        rows[part] = n < l.rows ? *reinterpret_cast<const v4i*>(g.state + n * g.state_words) : v4i{0, 0, 0, 0};
      }
#pragma unroll
      for (int part = 0; part < T::BJ; ++part) {
#pragma unroll
        for (int i = 0; i < T::BI; ++i) {
          const int it = (wi * T::BI + i) * 16 + 4 * (lane >> 4);
          out.put(wj * 16 + (lane & 15), it, grad_of(acc[i][part], rows[part], k, i0 + it, l.classes));
        }
        __syncthreads();
        if (part == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (see logit_tiles)
#pragma unroll
        for (int q = 0; q < kRows * Outgoing<T>::kPieces / T::kThreads; ++q) {
          const int at = q * T::kThreads + thread, r = at / Outgoing<T>::kPieces, c = at % Outgoing<T>::kPieces, nr = j0 + row_of(r, part);
          if (nr < l.rows && i0 + 8 * c < padded) *reinterpret_cast<v4i*>(g.g + nr * g.pitch + i0 + 8 * c) = *reinterpret_cast<const v4i*>(out.at(r, c));
        }
        __syncthreads();
      }
    });
  } else {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / T::WJ, wj = wave % T::WJ;
    int bi, bj;
    tile_of(blockIdx.x, ti, tj, &bi, &bj);
    const int i0 = bi * T::TI, j0 = bj * T::TJ;
    // what the end of the tile asks for goes out ahead of the products, where there are registers for it
    constexpr bool kEarly = T::RING > 1;
    const auto state_of = [&](int j) {
      const int n = j0 + (wj * T::BJ + j) * 16 + (lane & 15);
      return n < l.rows ? *reinterpret_cast<const v4i*>(g.state + n * g.state_words) : v4i{0, 0, 0, 0};
    };
    v4i rows[T::BJ];
    if constexpr (kEarly) {
#pragma unroll
      for (int j = 0; j < T::BJ; ++j) rows[j] = state_of(j);
    }
    const int places = min(T::TJ, l.rows - j0) * g.top;
    const auto place_of = [&](int at, int* j) {       // (gradient, class) of the tile's place `at`, which is row *j's
      *j = at / max(g.top, 1);
      return *reinterpret_cast<const int2*>(g.state + (j0 + *j) * g.state_words + 4 + 2 * (at - *j * g.top));
    };
    int2 place = make_int2(0, -1);
    int place_row = 0;
    if (kEarly && static_cast<int>(threadIdx.x) < places) place = place_of(threadIdx.x, &place_row);
    Sums<T, kFast, kFast, v4i> p;
    p.run(l.w, l.a, i0, j0, 0, (l.features + kStageBytes - 1) / kStageBytes, l.w.row_bytes, l.a.row_bytes, smem);
    const Outgoing<T> out{smem};
    if constexpr (!kEarly) {
#pragma unroll
      for (int j = 0; j < T::BJ; ++j) rows[j] = state_of(j);
    }
#pragma unroll
    for (int j = 0; j < T::BJ; ++j) {
#pragma unroll
      for (int i = 0; i < T::BI; ++i) {
        const int it = (wi * T::BI + i) * 16 + 4 * (lane >> 4);
        out.put((wj * T::BJ + j) * 16 + (lane & 15), it, grad_of(p.acc[i][j], rows[j], k, i0 + it, l.classes));
      }
    }
    __syncthreads();
    if (g.top > 0) {
      for (int at = threadIdx.x; at < places; at += T::kThreads) {
        if (!kEarly || at >= T::kThreads) place = place_of(at, &place_row);
        const long long i = place.y - g.first - i0;
        if (place.y >= 0 && i >= 0 && i < T::TI && i0 + i < l.classes) *out.one(place_row, static_cast<int>(i)) = target_grad(place.x);
      }
      __syncthreads();
    }
    for (int at = threadIdx.x; at < T::TJ * Outgoing<T>::kPieces; at += T::kThreads) {
      const int j = at / Outgoing<T>::kPieces, c = at % Outgoing<T>::kPieces;
      if (j0 + j < l.rows && i0 + 8 * c < padded) *reinterpret_cast<v4i*>(g.g + (j0 + j) * g.pitch + i0 + 8 * c) = *reinterpret_cast<const v4i*>(out.at(j, c));
    }
  }
}

__device__ inline uint16_t bf16_of(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }   // to nearest, ties to even

__device__ inline int sums_exponent(const VocabSums& s) { return *s.exponent + s.bias + (s.exponent2 != nullptr ? *s.exponent2 : 0); }
__device__ inline float sums_weight(const VocabSums& s, int j) { return s.weight == nullptr ? s.t : s.t * s.weight[s.weight_n == 1 ? 0 : j]; }

template <class T, Layout LX, Layout LY>
__device__ inline void sums_tile(const VocabSums& s, int block, char* smem) {
  const int ti = (s.ni + T::TI - 1) / T::TI, tj = (s.nj + T::TJ - 1) / T::TJ;
  const int slice = block / (ti * tj);
  if (slice >= s.slices) return;
  int bi, bj;
  tile_of(block - slice * ti * tj, ti, tj, &bi, &bj);
  const int i0 = bi * T::TI, j0 = bj * T::TJ;
  const int stages = (s.nk + 63) / 64;
  const int k0 = slice * s.steps;
  const int n = min(s.steps, stages - k0);
  const int end = min(s.nk, (k0 + n) * 64);      // steps
  const int e = sums_exponent(s);
  Sums<T, LX, LY, v4f> p;
  p.run(s.x, s.y, i0, j0, k0, n, LX == kFast ? 2 * ((end + 7) & ~7) : end, LY == kFast ? 2 * ((end + 7) & ~7) : end, smem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / T::WJ, wj = wave % T::WJ;
  if (s.part != nullptr) {
#pragma unroll
    for (int j = 0; j < T::BJ; ++j) {
      const int jj = j0 + (wj * T::BJ + j) * 16 + (lane & 15);
      if (jj >= s.nj) continue;
      float* const row = s.part + (static_cast<long long>(slice) * s.nj + jj) * s.part_pitch;
#pragma unroll
      for (int i = 0; i < T::BI; ++i) {
        const int ii = i0 + (wi * T::BI + i) * 16 + 4 * (lane >> 4);
        if (ii >= s.ni) continue;
        v4f* const at = reinterpret_cast<v4f*>(row + ii);
        v4f v = p.acc[i][j];
        if (s.accumulate) v += *at;
        *at = v;
      }
    }
    return;
  }
  const Outgoing<T> out{smem};
#pragma unroll
  for (int j = 0; j < T::BJ; ++j) {
    const int jt = (wj * T::BJ + j) * 16 + (lane & 15);
    const float weight = j0 + jt < s.nj ? sums_weight(s, j0 + jt) : 0.0f;
#pragma unroll
    for (int i = 0; i < T::BI; ++i) {
      uint64_t four = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) four |= static_cast<uint64_t>(bf16_of(ldexpf(p.acc[i][j][r] * weight, e))) << (16 * r);
      out.put(jt, (wi * T::BI + i) * 16 + 4 * (lane >> 4), four);
    }
  }
  __syncthreads();
  if ((s.ni & 7) == 0) {
    for (int at = threadIdx.x; at < T::TJ * Outgoing<T>::kPieces; at += T::kThreads) {
      const int j = at / Outgoing<T>::kPieces, c = at % Outgoing<T>::kPieces;
      if (j0 + j < s.nj && i0 + 8 * c < s.ni)
        *reinterpret_cast<v4i*>(s.out + static_cast<long long>(j0 + j) * s.ni + i0 + 8 * c) = *reinterpret_cast<const v4i*>(out.at(j, c));
    }
  } else {      // rows that start anywhere: whole sixteen bytes from the first multiple of sixteen on, then what is left at both ends
    const int width = min(T::TI, s.ni - i0), rows = min(T::TJ, s.nj - j0);
    const auto row_of = [&](int j) { return s.out + static_cast<long long>(j0 + j) * s.ni + i0; };
    const auto lead_of = [&](const uint16_t* row) { return min(width, static_cast<int>((-reinterpret_cast<intptr_t>(row) & 15) >> 1)); };
    for (int at = threadIdx.x; at < rows * Outgoing<T>::kPieces; at += T::kThreads) {
      const int j = at / Outgoing<T>::kPieces, c = at % Outgoing<T>::kPieces;
      uint16_t* const row = row_of(j);
      const int from = lead_of(row) + 8 * c;
      if (from + 8 > width) continue;
      v4i v;
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] = *out.one(j, from + 2 * d) | *out.one(j, from + 2 * d + 1) << 16;
      *reinterpret_cast<v4i*>(row + from) = v;
    }
    for (int at = threadIdx.x; at < rows * 16; at += T::kThreads) {      // up to seven values in front and behind
      const int j = at >> 4, e = at & 15;
      uint16_t* const row = row_of(j);
      const int lead = lead_of(row), behind = lead + (width - lead) / 8 * 8;
      const int i = e < 8 ? e : behind + e - 8;
      if (e < 8 ? i < lead : i < width) row[i] = *out.one(j, i);
    }
  }
}

// Bound by the products where rows are many: 8192 x 4096, 8192 classes 766 - 809 us for both (1.36 - 1.43 PFLOP/s; the library's product reaches
// 1.43), by memory where they are few: 31 x 4096 over 32000 70 us, 393 MB at 5.6 TB/s.  Sums of 32 bits; what is 16 bits wide on the way
// in has eleven significant ones.
// Both gradients' sums: the first `blocks_a` workgroups (a multiple of eight, see tile_of) the activations', the others the weights'.  The
// large tile reads a 16-bit copy of the int8 weights: made 16-bit in registers its fragments take 487 us of 8192 x 8192 x 4096, read from
// the copy 435, and the copy is 20 us of workgroups in the shadow of another launch.
template <class TA, class TW>
__global__ __launch_bounds__(TA::kThreads, TA::kPerUnit < TW::kPerUnit ? TA::kPerUnit : TW::kPerUnit) void vocab_sums_kernel(const VocabSums a, const VocabSums w, int blocks_a) {
  static_assert(TA::kThreads == TW::kThreads, "one launch");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  if (static_cast<int>(blockIdx.x) < blocks_a) sums_tile<TA, TA::TI == 256 ? kSlow16 : kSlow8, kFast>(a, blockIdx.x, smem);
  else sums_tile<TW, kSlow16, kSlow16>(w, blockIdx.x - blocks_a, smem);
}

// Adds the slices, scales, rounds (or leaves float32 as it is); a lane takes four neighbours of a row.  Bound by memory: 8192 x 4096 in one part
// 44 us, 201 MB at 4.6 TB/s
template <bool F32>
__device__ inline void join_block(const VocabSums& s, long long block) {
  const int quads = (s.ni + 3) / 4;
  const long long at = block * 256 + threadIdx.x, all = static_cast<long long>(quads) * s.nj;
  if (at >= all) return;
  const int j = static_cast<int>(all < 0x7fffffffLL ? static_cast<unsigned>(at) / static_cast<unsigned>(quads) : at / quads), i = static_cast<int>(at - static_cast<long long>(j) * quads) * 4;
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
  if constexpr (F32) {
    float* const out = s.out32 + static_cast<long long>(j) * s.ni + i;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r] * weight, e);
    if ((s.ni & 3) == 0) {
      *reinterpret_cast<v4f*>(out) = v;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (i + r < s.ni) out[r] = v[r];
    }
    return;
  }
  uint16_t* const out = s.out + static_cast<long long>(j) * s.ni + i;
  uint16_t b[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) b[r] = bf16_of(ldexpf(v[r] * weight, e));
  if ((s.ni & 3) == 0) {
    *reinterpret_cast<uint64_t*>(out) = b[0] | static_cast<uint64_t>(b[1]) << 16 | static_cast<uint64_t>(b[2]) << 32 | static_cast<uint64_t>(b[3]) << 48;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (i + r < s.ni) out[r] = b[r];
  }
}
template <bool F32>
__global__ __launch_bounds__(256) void vocab_join_kernel(const VocabSums a, const VocabSums w, int blocks_a) {
  if (static_cast<int>(blockIdx.x) < blocks_a) join_block<F32>(a, blockIdx.x);
  else join_block<F32>(w, blockIdx.x - blocks_a);
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

long long tiles_of(long long ni, long long nj, int ti, int tj) { return ((ni + ti - 1) / ti) * ((nj + tj - 1) / tj); }

// workgroups of a logits' launch: one per tile, or as many as the device holds at once
template <class T>
long long logit_blocks(const VocabLogits& l) {
  const long long tiles = tiles_of(l.classes, l.rows, T::TI, T::TJ), units = compute_units() / 8 * 8;
  return T::kInTurn && tiles > units ? units : tiles;
}
template <class T>
int run_stats(const VocabLogits& l, const VocabStats& s, const VocabTargets& targets, hipStream_t stream) {
  // beside the tiles they have the tiles' LDS, hence few wavefronts of a unit: many go out in a launch of their own
  const long long units = static_cast<long long>(l.rows) * ((targets.top + kPlaces - 1) / kPlaces);
  const bool apart = units > 4096;
  const long long dots = apart ? 0 : ((units + T::kWaves - 1) / T::kWaves + 7) / 8 * 8;
  const long long blocks = logit_blocks<T>(l) + dots;
  if (const int rc = check_grid(blocks, T::kThreads, "vocab_stats")) return rc;
  if (const int rc = check_grid((units + 3) / 4, 256, "vocab_dots")) return rc;
  if (tiles_of(l.classes, l.rows, T::TI, T::TJ) > 0x7fffffffLL) return fail(NITI_ERR_UNSUPPORTED, "vocab_stats: 2^31 tiles and more");
  if (const int rc = with_lds<vocab_stats_kernel<T>>(T::kLdsLogits, "vocab_stats")) return rc;
  if (apart) {
    hipLaunchKernelGGL(vocab_dots_kernel, dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), 0, stream, l, targets);
    if (const int rc = check_launch("vocab_dots")) return rc;
  }
  hipLaunchKernelGGL(vocab_stats_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(T::kThreads), T::kLdsLogits, stream, l, s, targets, static_cast<int>(dots));
  return check_launch("vocab_stats");
}
template <class T>
int run_grad(const VocabLogits& l, const VocabGrad& g, hipStream_t stream) {
  const long long blocks = logit_blocks<T>(l) + (g.widen_a.blocks + g.widen_w.blocks + 7) / 8 * 8;
  if (const int rc = check_grid(blocks, T::kThreads, "vocab_grad")) return rc;
  if (tiles_of(l.classes, l.rows, T::TI, T::TJ) > 0x7fffffffLL) return fail(NITI_ERR_UNSUPPORTED, "vocab_grad: 2^31 tiles and more");
  if (const int rc = with_lds<vocab_grad_kernel<T>>(T::kLdsLogits, "vocab_grad")) return rc;
  hipLaunchKernelGGL(vocab_grad_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(T::kThreads), T::kLdsLogits, stream, l, g);
  return check_launch("vocab_grad");
}
template <class TA, class TW>
int run_sums(const VocabSums& a, const VocabSums& w, hipStream_t stream) {
  constexpr int kLdsA = TA::kRings * TA::RING * (stage_bytes(TA::TI, TA::TI == 256 ? kSlow16 : kSlow8) + stage_bytes(TA::TJ, kFast)), kOutA = 2 * TA::TI * TA::TJ;
  constexpr int kMostA = kLdsA > kOutA ? kLdsA : kOutA, kLds = kMostA > TW::kLds ? kMostA : TW::kLds;
  const long long na = (tiles_of(a.ni, a.nj, TA::TI, TA::TJ) * a.slices + 7) / 8 * 8, nw = tiles_of(w.ni, w.nj, TW::TI, TW::TJ) * w.slices;
  if (const int rc = check_grid(na + nw, TA::kThreads, "vocab_sums")) return rc;
  if (const int rc = with_lds<vocab_sums_kernel<TA, TW>>(kLds, "vocab_sums")) return rc;
  hipLaunchKernelGGL((vocab_sums_kernel<TA, TW>), dim3(static_cast<unsigned>(na + nw)), dim3(TA::kThreads), kLds, stream, a, w, static_cast<int>(na));
  return check_launch("vocab_sums");
}

}  // namespace

// By statistics and gradients of 60 sizes (64 to 8192 rows, 512 to 100096 classes, 64 to 2048 features) with each tile.
//   Up to 32 rows, 64 x 32 and a stage for each wavefront where every tile has a unit and there is more than one stage for each:
//   30 x 2304 over 720 5.7 us (128 x 32 8.3), 1 x 4096 over 1000 7.2 (12.1), 16 x 1024 over 10000 5.1 (5.7), 2 x 128 over 64 4.0 (3.5)
//   64 x 64 and a stage for each wavefront likewise, the targets' workgroups beside the tiles counted: 100 x 4096 over 504 8.7 (64 x 64 together
//   11.0), 500 x 2304 over 1000 7.1 (7.9), 256 x 1536 over 4000, 252 tiles and 64, 8.2 (6.8)
//   64 x 64 where the device holds them all at once: 64 rows of 64 features over 20032 classes 4.4 us (128 x 128 4.9), of 2048 11 (16)
//   128 x 128 in a ring of two, two to a unit, where the device holds these at once and there are stages to overlap: 256 x 1024 over 10048 8.7
//   (one buffer and four to a unit 11.2), 256 x 256 5.6 (5.9), 256 x 64 5.0 (4.9)
//   256 x 256 in turn for long reductions on many rounds: a round is 1.68 of 128 x 128.  2048 x 2048 over 32064 141 (157), x 1024 79 (78), x 512 52 (48)
//   128 x 128 in one buffer, four to a unit, elsewhere: 1024 x 64 over 100096 41 (256 x 256 55, ring of two 60), 300 x 1024 over 30016 17 (22, 20)
VocabTile vocab_logits_tile(int rows, int features, int classes) {
  if (rows <= 32) return features >= 512 && tiles_of(classes, rows, 64, 32) <= 256 ? kVocabFewApart : kVocabFew;
  if (features > 1024 && tiles_of(classes, rows, 64, 64) + (rows + 3) / 4 <= 256) return kVocabSmallApart;
  if (tiles_of(classes, rows, 64, 64) <= 512) return kVocabSmall;
  const double middle = static_cast<double>(tiles_of(classes, rows, 128, 128)) / 512;
  if (middle <= 1.0) return features >= 512 ? kVocabMiddle : kVocabQuad;
  const double large = static_cast<double>((tiles_of(classes, rows, 256, 256) + 255) / 256);
  return features > 1024 && 1.68 * large <= middle ? kVocabLarge : kVocabQuad;
}

int vocab_stats_tiles(VocabTile t, int classes) {
  const bool narrow = t == kVocabSmall || t == kVocabSmallApart || t == kVocabFewApart;
  const int classes_of_tile = t == kVocabLarge ? TileLarge::TI : (narrow ? TileDeep::TI : TileMiddle::TI);
  static_assert(TileMiddle::TI == TileFew::TI && TileDeep::TI == TileFewApart::TI && TileDeep::TI == TileSmallApart::TI, "one rule");
  return (classes + classes_of_tile - 1) / classes_of_tile;
}

int launch_vocab_stats(VocabTile t, const VocabLogits& l, const VocabStats& s, const VocabTargets& targets, hipStream_t stream) {
  switch (t) {
    case kVocabLarge: return run_stats<TileLarge>(l, s, targets, stream);
    case kVocabMiddle: return run_stats<TileMiddle>(l, s, targets, stream);
    case kVocabSmall: return run_stats<TileDeep>(l, s, targets, stream);
    case kVocabQuad: return run_stats<TileShort>(l, s, targets, stream);
    case kVocabSmallApart: return run_stats<TileSmallApart>(l, s, targets, stream);
    case kVocabFewApart: return run_stats<TileFewApart>(l, s, targets, stream);
    default: return run_stats<TileFew>(l, s, targets, stream);
  }
}

bool vocab_sums_wants_wide_weights(VocabTile t) { return t == kVocabLarge; }

// a tile looks through the places of all of its rows: up to sixteen rounds of its threads.  Large ones have no registers for it
bool vocab_grad_writes_targets(VocabTile t, int top) { return t != kVocabLarge && top <= (t == kVocabFew || t == kVocabFewApart ? 128 : 32); }

int launch_vocab_grad(VocabTile t, const VocabLogits& l, const VocabGrad& g, hipStream_t stream) {
  switch (t) {
    case kVocabLarge: return run_grad<TileLarge>(l, g, stream);
    case kVocabMiddle: return run_grad<TileMiddle>(l, g, stream);
    case kVocabSmall: return run_grad<TileDeep>(l, g, stream);
    case kVocabQuad: return run_grad<TileShort>(l, g, stream);
    case kVocabSmallApart: return run_grad<TileSmallApart>(l, g, stream);
    case kVocabFewApart: return run_grad<TileFewApart>(l, g, stream);
    default: return run_grad<TileFew>(l, g, stream);
  }
}

namespace {
// What a workgroup of the sums takes, in us: per stage and beside them, with as many of its kind on the device as `slots`.  Fitted, with
// the two terms of the parts' adding below, to the times of every tile and cut for 35 sizes (1 to 8192 rows, 64 to 4096 features, 100 to 60032
// classes, some 1400 combinations): for those sizes what the plan picks is at most 4 % off the best of them.  The wavefronts' own stages (the two ...Apart)
// were fitted later, to 26 sizes of 1 to 400 rows, most within 10 % of the best: 16 x 512 over 2000 7.6 us (128 x 32 13.6), 128 x 512 over 1000 7.0 (8.7), but
// 32 x 64 over 4000 10.8 for 7.8.
struct SumsCost {
  int ti, tj, slots;
  double stage, fixed;
};
struct SumsCosts {
  VocabTile tile;
  int rows_from, rows_to;
  SumsCost a, w;
};
constexpr SumsCosts kSumsCosts[] = {
    {kVocabLarge, 33, 0x7fffffff, {256, 256, 256, 1.3, 6.0}, {256, 256, 256, 1.14, 8.4}},
    {kVocabMiddle, 33, 0x7fffffff, {128, 128, 512, 0.85, 5.5}, {128, 128, 512, 0.85, 4.0}},
    {kVocabQuad, 33, 0x7fffffff, {128, 128, 1024, 1.4, 6.0}, {128, 128, 1024, 1.2, 6.0}},
    {kVocabSmall, 33, 0x7fffffff, {64, 64, 1024, 0.7, 3.7}, {64, 64, 1024, 0.84, 3.0}},
    {kVocabShort, 33, 512, {64, 64, 1024, 0.61, 2.85}, {128, 128, 1024, 1.2, 6.8}},
    {kVocabSmallApart, 33, 512, {64, 64, 256, 0.25, 4.2}, {128, 128, 256, 1.2, 3.4}},
    {kVocabFewApart, 1, 32, {64, 32, 256, 0.11, 3.9}, {128, 128, 256, 1.0, 3.5}},
    {kVocabFew, 1, 32, {128, 32, 1024, 0.24, 3.0}, {128, 128, 1024, 1.0, 1.9}},
};
}  // namespace

// The tiles and cuts whose estimated time is least: all workgroups' time over the device's slots and a part of the longest one's, and the adding
// of the parts.
VocabTile vocab_sums_plan(int rows, int features, int classes, int* slices_a, int* steps_a, int* slices_w, int* steps_w) {
  const int sa = (classes + 63) / 64, sw = (rows + 63) / 64;
  const auto join = [features](int slices, long long nj) { return slices > 1 ? 7.7 + slices * 8.0 * features * static_cast<double>(nj) / 2.8e6 : 0.0; };
  VocabTile best_tile = kVocabLarge;
  double best = -1.0;
  for (const SumsCosts& c : kSumsCosts) {
    if (rows < c.rows_from || rows > c.rows_to) continue;
    const long long na = tiles_of(features, rows, c.a.ti, c.a.tj), nw = tiles_of(features, classes, c.w.ti, c.w.tj);
    for (int ca = 1; ca == 1 || (ca <= 64 && (sa + ca - 1) / ca >= 4); ca += (ca + 1) / 2) {
      const int step_a = (sa + ca - 1) / ca, na_cut = (sa + step_a - 1) / step_a;
      for (int cw = 1; cw == 1 || (cw <= 64 && (sw + cw - 1) / cw >= 4); cw += (cw + 1) / 2) {
        const int step_w = (sw + cw - 1) / cw, nw_cut = (sw + step_w - 1) / step_w;
        const double each_a = step_a * c.a.stage + c.a.fixed, each_w = step_w * c.w.stage + c.w.fixed;
        const double all = na * na_cut * each_a / c.a.slots + nw * nw_cut * each_w / c.w.slots, longest = each_a > each_w ? each_a : each_w;
        const double spread = all + 0.27 * longest;
        const double t = (spread > longest ? spread : longest) + join(na_cut, rows) + join(nw_cut, classes);
        if (best < 0.0 || t < best) {
          best = t;
          best_tile = c.tile;
          *slices_a = na_cut;
          *steps_a = step_a;
          *slices_w = nw_cut;
          *steps_w = step_w;
        }
      }
    }
  }
  return best_tile;
}

int launch_vocab_sums(VocabTile t, const VocabSums& a, const VocabSums& w, hipStream_t stream) {
  switch (t) {
    case kVocabLarge: return run_sums<TileLarge, TileLarge>(a, w, stream);
    case kVocabMiddle: return run_sums<TileMiddle, TileMiddle>(a, w, stream);
    case kVocabSmall: return run_sums<TileSmall, TileSmall>(a, w, stream);
    case kVocabShort: return run_sums<TileSmall, TileShort>(a, w, stream);
    case kVocabQuad: return run_sums<TileShort, TileShort>(a, w, stream);
    case kVocabSmallApart: return run_sums<TileSmallApart, TileShort>(a, w, stream);
    case kVocabFewApart: return run_sums<TileFewApart, TileShort>(a, w, stream);
    default: return run_sums<TileFewSums, TileShort>(a, w, stream);
  }
}

int launch_vocab_join(const VocabSums* a, const VocabSums* w, hipStream_t stream) {
  const auto blocks = [](const VocabSums* s) { return s == nullptr ? 0 : (static_cast<long long>((s->ni + 3) / 4) * s->nj + 255) / 256; };
  const long long na = blocks(a), nw = blocks(w);
  if (const int rc = check_grid(na + nw, 256, "vocab_join")) return rc;
  const auto kernel = (a != nullptr ? a : w)->out32 != nullptr ? vocab_join_kernel<true> : vocab_join_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(na + nw)), dim3(256), 0, stream, a != nullptr ? *a : *w, w != nullptr ? *w : *a, static_cast<int>(na));
  return check_launch("vocab_join");
}

}  // namespace niti
