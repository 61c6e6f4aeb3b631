// libvsloss.so -- softmax cross entropy of z = hidden weight^T + bias, forward and backward, in pieces of the vocabulary:
//
//   forward    z tile by tile on the matrix cores; each tile leaves the maximum and the sum of exponentials of its classes
//              for every row, and the target's logit; a small kernel joins them into lse and the row losses.
//   backward   for a piece of the vocabulary: z again, d = g (p (1 + 2 z_loss lse) - [class == target]) rounded to the
//              operands' type and written as [rows, piece] and as [piece, rows]; then
//              grad_hidden += d weight_piece (float32 across the pieces) and grad_weight_piece = d^T hidden.
//
// d is rounded because a second plane for the rest of it would double both gradient products and the derivatives' traffic.
// Gradients that are rounded to 16 bits at the end lose little by it: off against float64 by 1.8e-3 of their size instead of
// 1.7e-3 (8192 x 131072 x 4096 bfloat16), 4.1e-4 instead of 3.8e-4 (2011 x 32003 x 1000 float16), 2.2e-3 instead of 1.7e-3
// (92160 x 128 x 256 bfloat16).
//
// All three products are C[M,N] = A[M,K] B[N,K]^T with K contiguous in both operands, so that one main loop serves them:
// the transposed weight and hidden that the two gradient products need are laid out once per call.  Recomputing z costs
// a fourth product (a third more operations than keeping the logits) and spares rows * vocab float32 of memory traffic.
//
// Float32 has two forms.  The direct one uses the float32 matrix instructions (105 TFLOP/s here).  The split one writes
// every float as the sum of three bfloat16, x = h + m + l, which holds all of its 24 bits, and multiplies
// x y = l h + m m + h l + m h + h m + h h; what it leaves out (m l, l m, l l) is below 2^-24 of the product, as a float32
// product's own rounding is, and the sums stay float32.  Six bfloat16 products run 2.7 times faster than one float32
// product; their operands are laid out as three planes per row, and the main loop walks the six pairs of planes one after
// the other, smallest first.
#include <algorithm>
#include <type_traits>

#include "vsl_vocab.hpp"

namespace vsl_vocab {
namespace {

static_assert(sizeof(vsl_linear_ce_desc) == 96, "C-ABI struct layout changed");

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;    // of the kernels around the products
constexpr int kBlockBytes = 128; // bytes of K that one step of the main loop takes from every row of A and B
constexpr int kPad = 256;        // rows and classes are laid out in multiples of the larger tile

// Shape of an output tile: BM x BN, WM x WN waves, each with IM x JN blocks of 32 x 32.
template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int IM = BM / WM / 32, JN = BN / WN / 32;
  static constexpr int kBuffer = (BM + BN) * kBlockBytes;  // LDS of one step
  static constexpr int kLds = 2 * kBuffer;
  static constexpr int kFetch = kBuffer / (kThreads * 16);  // 16-byte pieces per thread and step, A's first
  static constexpr int kFetchA = BM * kBlockBytes / (kThreads * 16);
};
typedef Shape<256, 256, 2, 4> Large;
typedef Shape<128, 128, 2, 2> Small;
typedef Shape<128, 64, 4, 1> Narrow;  // few columns: rows of the loss
typedef Shape<128, 32, 4, 1> Thin;    // 32 at most

template <typename T>
struct Kind {
  static constexpr int E = 16 / (int)sizeof(T);             // elements of a 16-byte piece
  static constexpr int BK = kBlockBytes / (int)sizeof(T);   // elements of K per step
};

// One 16-byte piece of A (row = lane % 32) and of B (column = lane % 32) per lane; the two halves of the wave hold
// neighbouring pieces of K.  Float32 takes the four elements of a piece one after the other: which K meet in one
// instruction does not matter as long as A and B agree.
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c, const __bf16*) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c, const _Float16*) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c, const float*) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
  return c;
}

// 16 bytes of a row that may start anywhere, zeros behind the last column
template <typename T>
__device__ __forceinline__ u32x4 load_columns(const T* p, int c, int cols) {
  if (c + Kind<T>::E <= cols) return load16(p + c);
  float v[Kind<T>::E];
#pragma unroll
  for (int e = 0; e < Kind<T>::E; ++e) v[e] = c + e < cols ? (float)p[c + e] : 0.0f;
  return pack(v, (const T*)nullptr);
}
// Operands of a product: A [M, >= kblocks * BK], B [N, ...], rows `lda`, `ldb` elements apart; in the split form the
// planes of a row are plane_a, plane_b elements apart.
struct Operands {
  const void* A;
  const void* B;
  int64_t lda, ldb;
  int M, N, kblocks;
  int64_t plane_a, plane_b;
  int tail;  // 16-byte pieces of a row in the last block (8: it is whole); what follows them is not the row's
  int dim;   // elements of a row, where rows lie at any address (kStagedRows)
  int rows_of_k;     // kStagedColumns: rows of A
  const void* bias;  // kStagedColumns: rows of A at -infinity here count as zeros, or NULL
};
enum { kDirect, kStagedRows, kStagedColumns };  // ways of the operands to LDS
// what the pieces behind a row's end are read from
__device__ const u32x4 kZeros[1] = {{0u, 0u, 0u, 0u}};
constexpr int kPairs = 6;
// planes of pair p, two bits each: l h, m m, h l, m h, h m, h h (h = 0, m = 1, l = 2)
__device__ __forceinline__ int pair_a(int p) { return (0x046 >> (2 * p)) & 3; }
__device__ __forceinline__ int pair_b(int p) { return (0x124 >> (2 * p)) & 3; }

// C tile of a wave: acc[i][j] covers rows 32 i.. and columns 32 j.. of its part; register r of a lane is row
// (r & 3) + 8 (r >> 2) + 4 (lane >> 5), column lane & 31.
template <typename S>
struct Tile {
  f32x16 acc[S::IM][S::JN];
};

// Rows of A and B go through LDS 128 bytes at a time, two buffers deep, straight from global memory.  A row is one line
// of eight 16-byte pieces; piece p of row r lies at p ^ ((r >> 1) & 7), so that sixteen rows read at one
// piece touch all 64 banks (with r & 7 half of the reads' cycles were conflicts).
// A step is four rounds; each round's fragments are read while the round before multiplies.  The barrier stands before the
// last round, whose fragments are in registers by then: behind it the buffer is free for the step after next, and the
// next step's first fragments are read under the last round's multiplications.
// kStagedRows: rows that start anywhere or end inside a piece cannot go straight to LDS.  They go through registers, asked for
// a step ahead of their store, which takes the place of the fetch.
// kStagedColumns: so does an A that lies as [K, M]: BM elements of every row of a step, whose fragments are gathered from LDS
// element by element; the two halves of the wave, E rows apart, read 32 elements apart as well, from other banks.
// T: the operands' type; steps [k0, k1) of kblocks, or of kPairs * kblocks in the split form.
template <typename T, typename S, bool SPLIT, int FORM>
__device__ __forceinline__ void tile_product(const Operands& op, int m0, int n0, int k0, int k1, char* lds, Tile<S>& t) {
  constexpr bool STAGED = FORM != kDirect, COLUMNS = FORM == kStagedColumns;
  constexpr int E = Kind<T>::E, kWide = S::BM / E;  // COLUMNS: pieces of A's BM elements of a row
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int i = 0; i < S::IM; ++i)
#pragma unroll
    for (int j = 0; j < S::JN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) t.acc[i][j][r] = 0.0f;
  if (k0 >= k1) return;
  const char* src[S::kFetch];
  int pair = 0, at_k = k0;
  int64_t offset_a = (int64_t)k0 * kBlockBytes, offset_b = offset_a;
  if (SPLIT) {
    pair = k0 / op.kblocks;
    at_k = k0 - pair * op.kblocks;
    offset_a = pair_a(pair) * op.plane_a * (int)sizeof(T) + (int64_t)at_k * kBlockBytes;
    offset_b = pair_b(pair) * op.plane_b * (int)sizeof(T) + (int64_t)at_k * kBlockBytes;
  }
#pragma unroll
  for (int i = 0; i < S::kFetch; ++i) {
    const int at = (i < S::kFetchA ? i : i - S::kFetchA) * S::kThreads + tid, row = at >> 3, piece = (at & 7) ^ ((row >> 1) & 7);
    src[i] = i < S::kFetchA ? (const char*)op.A + (int64_t)min(m0 + row, op.M - 1) * op.lda * (int)sizeof(T)
                            : (const char*)op.B + (int64_t)min(n0 + row, op.N - 1) * op.ldb * (int)sizeof(T);
    src[i] += (i < S::kFetchA ? offset_a : offset_b) + piece * 16;
  }
  int left = k1 - k0;  // steps to fetch
  auto fetch = [&](int buffer) {
    if (!SPLIT && --left == 0 && k1 == op.kblocks && op.tail < 8) {
#pragma unroll
      for (int i = 0; i < S::kFetch; ++i) {
        const int at = (i < S::kFetchA ? i : i - S::kFetchA) * S::kThreads + tid;
        if (((at & 7) ^ ((at >> 4) & 7)) >= op.tail) src[i] = (const char*)kZeros;
      }
    }
    int64_t next_a = kBlockBytes, next_b = kBlockBytes;
    if (SPLIT && ++at_k == op.kblocks) {  // on to the next pair of planes, from its beginning
      const int64_t back = (int64_t)(op.kblocks - 1) * kBlockBytes;
      next_a = (pair_a(pair + 1) - pair_a(pair)) * op.plane_a * (int)sizeof(T) - back;
      next_b = (pair_b(pair + 1) - pair_b(pair)) * op.plane_b * (int)sizeof(T) - back;
      at_k = 0;
      ++pair;
    }
#pragma unroll
    for (int i = 0; i < S::kFetch; ++i) {
      char* dst = lds + buffer * S::kBuffer + (i * S::kThreads + wave * 64) * 16;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src[i],
                                       (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
      src[i] += i < S::kFetchA ? next_a : next_b;
    }
  };
  u32x4 held[STAGED ? S::kFetch : 1];
  int next_step = k0;
  auto load = [&]() {
    const int first = next_step * Kind<T>::BK + ((tid & 7) ^ ((tid >> 4) & 7)) * Kind<T>::E;  // column of a thread's pieces
    const bool whole = (++next_step) * Kind<T>::BK <= op.dim;
    // a piece that runs over the end of its row reads on in the next one (of 8 elements or more): those columns of the tile
    // are nobody's
    const bool followed = COLUMNS && next_step * Kind<T>::BK < op.rows_of_k;
#pragma unroll
    for (int i = 0; i < (STAGED ? S::kFetch : 0); ++i) {
      if (COLUMNS && i < S::kFetchA) {
        const int at = i * S::kThreads + tid, k = at / kWide, row = (next_step - 1) * Kind<T>::BK + k;
        const int m = m0 + (at % kWide * E ^ (k / E & 1) * 32);
        if (followed) {
          held[i] = load16((const T*)op.A + (int64_t)row * op.lda + min(m, op.M - 1));
        } else {
          held[i] = u32x4{0u, 0u, 0u, 0u};
          if (row < op.rows_of_k) held[i] = load_columns((const T*)op.A + (int64_t)row * op.lda, m, op.M);
        }
      } else {
        held[i] = COLUMNS || whole ? load16((const T*)src[i]) : load_columns((const T*)src[i], 0, op.dim - first);
        src[i] += kBlockBytes;
      }
    }
  };
  auto store = [&](int buffer) {
    if (COLUMNS && op.bias)  // rows of the step that is held
#pragma unroll
      for (int i = 0; i < S::kFetchA; ++i) {
        const int row = (next_step - 1) * Kind<T>::BK + (i * S::kThreads + tid) / kWide;
        if ((float)((const T*)op.bias)[min(row, op.rows_of_k - 1)] == ninf()) held[i] = u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
    for (int i = 0; i < (STAGED ? S::kFetch : 0); ++i) *(u32x4*)(lds + buffer * S::kBuffer + (i * S::kThreads + tid) * 16) = held[i];
  };
  auto wait = [&]() {  // this wave's pieces are in LDS and its reads are done; then everyone's are
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  const char* a = lds + (wm * S::IM * 32 + (lane & 31)) * kBlockBytes;
  const char* b = lds + (S::BM + wn * S::JN * 32 + (lane & 31)) * kBlockBytes;
  u32x4 fa[2][S::IM], fb[2][S::JN];
  auto read = [&](int set, int buffer, int round) {
    const int piece = ((2 * round + (lane >> 5)) ^ ((lane >> 1) & 7)) * 16 + buffer * S::kBuffer;
    if constexpr (COLUMNS) {
      const T* column = (const T*)(lds + buffer * S::kBuffer) + (2 * round + (lane >> 5)) * E * S::BM;
#pragma unroll
      for (int i = 0; i < S::IM; ++i) {
        const int m = ((wm * S::IM + i) * 32 + (lane & 31)) ^ (lane & 32);
        union {
          T t[E];
          u32x4 u;
        } f;
#pragma unroll
        for (int e = 0; e < E; ++e) f.t[e] = column[e * S::BM + m];
        fa[set][i] = f.u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < S::IM; ++i) fa[set][i] = *(const u32x4*)(a + i * 32 * kBlockBytes + piece);
    }
#pragma unroll
    for (int j = 0; j < S::JN; ++j) fb[set][j] = *(const u32x4*)(b + j * 32 * kBlockBytes + piece);
  };
  auto multiply = [&](int set) {
#pragma unroll
    for (int i = 0; i < S::IM; ++i)
#pragma unroll
      for (int j = 0; j < S::JN; ++j) t.acc[i][j] = mma(fa[set][i], fb[set][j], t.acc[i][j], (const T*)nullptr);
  };
  auto interleave = [&]() {  // a round's reads go out one by one behind its multiplications, and stay in their round
    constexpr int kMma = S::IM * S::JN * (sizeof(T) == 4 ? 4 : 1), kRead = S::IM + S::JN;
    constexpr int kEach = kMma / (kRead + 2) < 1 ? 1 : kMma / (kRead + 2);
    if (COLUMNS) return;  // bound by its reads of A from memory
#pragma unroll
    for (int i = 0; i < kRead; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kMma - kRead * kEach, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  if (STAGED) {
    load();
    store(0);
    if (k0 + 1 < k1) load();
  } else {
    fetch(0);
  }
  wait();
  if (k0 + 1 < k1) STAGED ? store(1) : fetch(1);
  read(0, 0, 0);
  auto rounds = [&](int buffer) {  // the first three
#pragma unroll
    for (int round = 0; round < 3; ++round) {
      read((round + 1) & 1, buffer, round + 1);
      multiply(round & 1);
      interleave();
    }
  };
  for (int k = k0; k < k1 - 1; ++k) {
    const int buffer = (k - k0) & 1;
    if (STAGED && k + 2 < k1) load();
    rounds(buffer);
    wait();
    if (k + 2 < k1) STAGED ? store(buffer) : fetch(buffer);
    read(0, buffer ^ 1, 0);
    multiply(1);
    interleave();
  }
  rounds((k1 - 1 - k0) & 1);
  multiply(1);
  __syncthreads();
}

// Workgroups are dealt to the 8 XCDs in turn; every XCD gets a contiguous run of tiles, walked in columns of eight rows of
// tiles, so that the operands' panels meet in one L2.
__device__ __forceinline__ void tile_of(int64_t block, int64_t tiles_m, int64_t tiles_n, int& tm, int& tn) {
  const int64_t n = tiles_m * tiles_n, per = n / 8, extra = n % 8, xcd = block % 8;
  const int64_t i = xcd * per + min(xcd, extra) + block / 8;
  const int64_t group = 8 * tiles_n, first = i / group * 8, height = min((int64_t)8, tiles_m - first);
  tm = (int)(first + i % group % height);
  tn = (int)(i % group / height);
}

// ------------------------------------------------------------------------------------------------------------------
// forward: A = weight (rows of C are classes), B = hidden (columns are rows of the loss)
// ------------------------------------------------------------------------------------------------------------------
struct LogitArgs {
  Operands op;
  // float32 by planes: the operands as they were given
  const float *given_a, *given_b;
  int64_t given_lda, given_ldb;
  const void* bias;
  const int64_t* target;
  int64_t class0;      // first class of the piece
  int64_t rows_padded;
  // forward
  float2* partial;     // [tiles_m][rows_padded] maximum and sum
  float* target_logit; // [rows]
  // backward
  const float* stats;  // [2][rows] maximum and log2 of the sum above it
  const float* row_scale;  // kRowDerivatives; otherwise `unit` for every row that counts
  const float* row_size;   // what the row's scale was divided by; out_scale: the largest of them
  const float* out_scale;
  float unit;
  int64_t ignore_index;
  float z_loss;
  void* delta;         // [rows_padded][ldd], planes plane_d apart
  int64_t ldd, plane_d;
  void* delta_t;       // [padded classes of the piece][ldt], planes rows_padded apart
  int64_t ldt;
};

// Adds the biases of a block's classes, which lie in LDS as floats, -infinity behind the last class.
__device__ __forceinline__ void add_bias(f32x16& z, const float* bias) {
#pragma unroll
  for (int r4 = 0; r4 < 4; ++r4) {
    const f32x4 b = *(const f32x4*)(bias + 8 * r4);
#pragma unroll
    for (int e = 0; e < 4; ++e)  // a masked class stays masked whatever its weights hold
      z[4 * r4 + e] = b[e] == ninf() ? b[e] : z[4 * r4 + e] + b[e];
  }
}

// derivative of lse + z_loss lse^2 with respect to lse
__device__ __forceinline__ float slope_of(float z_loss, float top, float ls) {
  return z_loss == 0.0f ? 1.0f : fmaf(2.0f * z_loss, fmaf(ls, kLn2, top), 1.0f);
}

// Four 16-bit values a lane, of four lanes in a row, transposed: lane q of the four ends with value q of each.
__device__ __forceinline__ uint2 transpose4(uint2 x) {
  const unsigned q = threadIdx.x & 3;
  const unsigned got = dpp<kXor2>(q < 2 ? x.y : x.x);
  const unsigned a = q < 2 ? x.x : got, b = q < 2 ? got : x.y;  // values 2 (q / 2).. of lanes q & 1 and (q & 1) + 2
  const unsigned lows = (a & 0xFFFFu) | b << 16, highs = a >> 16 | (b & 0xFFFF0000u);
  const unsigned other = dpp<kXor1>(q & 1 ? lows : highs);
  const unsigned even = q & 1 ? other : lows, odd = q & 1 ? highs : other;  // lanes 0, 2 and lanes 1, 3
  return {(even & 0xFFFFu) | odd << 16, even >> 16 | (odd & 0xFFFF0000u)};
}
template <typename T>
__device__ __forceinline__ uint2 pack4(const float (&g)[4]) {
  union {
    T t[4];
    uint2 u;
  } p;
#pragma unroll
  for (int e = 0; e < 4; ++e) p.t[e] = (T)g[e];
  return p.u;
}

// z -> its part that bfloat16 holds, and what is left of it
__device__ __forceinline__ float take_plane(float& z) {
  const float h = (float)(__bf16)z;
  z -= h;
  return h;
}

// Logits by planes that are not finite are made again from the floats themselves: an infinity has no planes (what is left of it
// is infinity minus infinity), and a logit of -infinity is a masked class however its product was formed.  A wave makes its own,
// four classes of 32 rows in either half at a time as sixteen products of 4 x 4, whose four registers are those of four classes in
// the tile; larger products would not fit beside the tile.  The fragments come straight from memory, at some hundredths of the
// direct form's rate.  Finite logits keep their bits, so that no row feels another's; those of masked classes and of rows that
// do not count are left as they are.
template <typename S>
__device__ __forceinline__ void exact_if_not_finite(const LogitArgs& a, int m0, int n0, Tile<S>& t) {
  float probe[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < S::IM; ++i)
#pragma unroll
    for (int j = 0; j < S::JN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) probe[r & 1] = fmaf(t.acc[i][j][r], 0.0f, probe[r & 1]);
  if (!__any(probe[0] + probe[1] != 0.0f)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int i = 0; i < S::IM; ++i)
#pragma unroll
    for (int j = 0; j < S::JN; ++j)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        bool wrong[4], any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= wrong[e] = t.acc[i][j][4 * r4 + e] * 0.0f != 0.0f;
        if (!__any(any)) continue;
        int m = m0 + (wm * S::IM + i) * 32 + 8 * r4 + 4 * (lane >> 5) + (lane & 3), n = n0 + (wn * S::JN + j) * 32 + (lane & 31);
        const bool masked = m >= a.op.M || (a.bias && ((const float*)a.bias)[a.class0 + m] == ninf());
        const bool counts = n < a.op.N && a.target[n] != a.ignore_index;
        any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= wrong[e] = wrong[e] && counts && !__shfl((int)masked, (lane & 32) + e, 64);
        if (!__any(any)) continue;
        asm volatile("" : "+v"(m), "+v"(n));  // addresses of these classes alone: made for all in advance they would spill
        const float* pa = a.given_a + (int64_t)min(m, a.op.M - 1) * a.given_lda;
        const float* pb = a.given_b + (int64_t)min(n, a.op.N - 1) * a.given_ldb;
        f32x4 z{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < a.op.dim && __any(any);) {  // until all are NaN, if they become that
          const int end = min(k + 64, a.op.dim);
          for (; k < end; ++k) z = __builtin_amdgcn_mfma_f32_4x4x1f32(pa[k], pb[k], z, 0, 0, 0);
          any = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) any |= wrong[e] && z[e] == z[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (wrong[e]) t.acc[i][j][4 * r4 + e] = z[e];
      }
}

enum { kStatistics, kDerivatives, kRowDerivatives };  // of the logits; derivatives of one gradient, or of one per row
// T: the tensors' type; SPLIT: float32 by planes of bfloat16.  8192 x 131072 x 4096 bfloat16: forward 6.98 ms, 1260 TFLOP/s,
// derivatives 8 x 1.01 ms, 1089; bound by the matrix instructions at the power the card allows, then by the epilogue's
// exponentials, which no other tile's products cover (a large tile fills its CU).  2011 x 32003 x 1000 float16: 149 and 187 us.
template <typename T, typename S, int WHAT, bool SPLIT, int FORM>
__global__ __launch_bounds__(S::kThreads) void k_ce_logits(LogitArgs a) {
  constexpr bool DELTA = WHAT != kStatistics, ROWS = WHAT == kRowDerivatives;
  typedef std::conditional_t<SPLIT, __bf16, T> O;
  __shared__ __attribute__((aligned(16))) char lds[S::kLds];
  const int tm_count = (a.op.M + S::BM - 1) / S::BM, tn_count = (a.op.N + S::BN - 1) / S::BN;
  int tm, tn;
  tile_of(blockIdx.x, tm_count, tn_count, tm, tn);
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  Tile<S> t;
  tile_product<O, S, SPLIT, FORM>(a.op, m0, n0, 0, (SPLIT ? kPairs : 1) * a.op.kblocks, lds, t);
  if constexpr (SPLIT) exact_if_not_finite<S>(a, m0, n0, t);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  const int half = lane >> 5;
  const bool biased = a.bias || m0 + S::BM > a.op.M;
  float* bias = (float*)(lds + S::WM * S::BN * sizeof(float2));
  if (biased) {
    for (int i = threadIdx.x; i < S::BM; i += S::kThreads)
      bias[i] = m0 + i >= a.op.M ? ninf() : a.bias ? (float)((const T*)a.bias)[a.class0 + m0 + i] : 0.0f;
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < S::JN; ++j) {
    const int col = (wn * S::JN + j) * 32 + (lane & 31), row = n0 + col;
    const bool live = row < a.op.N;
    const int64_t target = live ? a.target[row] - a.class0 : -1;
    // Most of an epilogue's elements are neither behind the last class nor a target: both are looked for once per 32
    // classes (16 of them in a lane's registers).
    if (!DELTA) {
      float m = ninf();
#pragma unroll
      for (int i = 0; i < S::IM; ++i) {
        const int v32 = m0 + (wm * S::IM + i) * 32;
        f32x16& z = t.acc[i][j];
        if (biased) add_bias(z, bias + v32 - m0 + 4 * half);
        if (target >= v32 && target < v32 + 32) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (v32 + (r & 3) + 8 * (r >> 2) + 4 * half == target) a.target_logit[row] = z[r];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) m = __builtin_elementwise_maximum(m, z[r]);
      }
      const Exponent ex(exp_ref(m), kLog2e);
      float s = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int i = 0; i < S::IM; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          s += ex(t.acc[i][j][r]);
          s2 += ex(t.acc[i][j][r + 1]);
        }
      MaxSum q{m, (s + s2) * ex.factor()};
      q = join(q, {__shfl_xor(q.m, 32, 64), __shfl_xor(q.s, 32, 64)}, kLog2e);
      if (half == 0) ((float2*)lds)[wm * S::BN + col] = make_float2(q.m, q.s);
    } else {
      const float top = live ? a.stats[row] : ninf(), ls = live ? a.stats[a.op.N + row] : 0.0f;
      const float scale = !live || top == ninf() || target + a.class0 == a.ignore_index ? 0.0f
                          : ROWS ? a.row_scale[row] : a.unit;
      const Exponent ex(top, kLog2e);
      const float factor = scale * slope_of(a.z_loss, top, ls) * ex.factor(ls);
      const float ratio = ROWS && live ? a.row_size[row] / *a.out_scale : 1.0f;  // a power of two
      O* d = (O*)a.delta + (int64_t)row * a.ldd;
#pragma unroll
      for (int i = 0; i < S::IM; ++i) {
        const int v32 = m0 + (wm * S::IM + i) * 32;
        f32x16& z = t.acc[i][j];
        if (biased) add_bias(z, bias + v32 - m0 + 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = factor * ex(z[r]);
        if (target >= v32 && target < v32 + 32) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (v32 + (r & 3) + 8 * (r >> 2) + 4 * half == target) z[r] -= scale;
        }
        if (scale == 0.0f) {  // whatever the row holds
#pragma unroll
          for (int r = 0; r < 16; ++r) z[r] = 0.0f;
        }
#pragma unroll
        for (int r8 = 0; r8 < 2; ++r8) {  // two groups of 8 classes, four of each in either half of the wave
          if constexpr (sizeof(O) == 4) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int v0 = v32 + 16 * r8 + 8 * u + 4 * half, r = 8 * r8 + 4 * u;
              if (a.delta) *(f32x4*)(d + v0) = f32x4{z[r], z[r + 1], z[r + 2], z[r + 3]};
              if (a.delta_t)
#pragma unroll
                for (int e = 0; e < 4; ++e) ((O*)a.delta_t)[(int64_t)(v0 + e) * a.ldt + row] = z[r + e] * ratio;
            }
          } else {
#pragma unroll
            for (int plane = 0; plane < (SPLIT ? 3 : 1); ++plane) {
              float g[2][4];
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float rest = z[8 * r8 + 4 * u + e];
                  g[u][e] = SPLIT ? take_plane(rest) : rest;
                  z[8 * r8 + 4 * u + e] = rest;
                }
              const uint2 p0 = pack4<O>(g[0]), p1 = pack4<O>(g[1]);
              if (a.delta) {
                // the halves trade: the lower lanes get all 8 classes of the first group, the upper ones those of the second
                const auto x = __builtin_amdgcn_permlane32_swap(p0.x, p1.x, false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(p0.y, p1.y, false, false);
                *(u32x4*)(d + plane * a.plane_d + v32 + 16 * r8 + 8 * half) = u32x4{x[0], y[0], x[1], y[1]};
              }
              if (a.delta_t) {
                uint2 t[2] = {p0, p1};
                if (ROWS) {
#pragma unroll
                  for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) g[u][e] *= ratio;
                    t[u] = pack4<O>(g[u]);
                  }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const int v = v32 + 16 * r8 + 8 * u + 4 * half + (lane & 3);
                  *(uint2*)((O*)a.delta_t + (int64_t)v * a.ldt + plane * a.rows_padded + (row & ~3)) = transpose4(t[u]);
                }
              }
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);  // blocks one after the other: mixed they need more registers than there are
      }
    }
  }
  if (!DELTA) {
    __syncthreads();
    const int col = threadIdx.x;
    if (col < S::BN) {
      float2 x = ((float2*)lds)[col];
      MaxSum q{x.x, x.y};
#pragma unroll
      for (int w = 1; w < S::WM; ++w) {
        x = ((float2*)lds)[w * S::BN + col];
        q = join(q, {x.x, x.y}, kLog2e);
      }
      a.partial[(int64_t)tm * a.rows_padded + n0 + col] = make_float2(q.m, q.s);
    }
  }
}

// A row's loss and statistics from its joined maximum and sum; logit(t): the target's.
template <typename F>
__device__ __forceinline__ float close_row(MaxSum q, F logit, int64_t t, int64_t ignore_index, int64_t vocab, float z_loss,
                                           int64_t row, int64_t rows, float* row_loss, float* stats, bool& counts) {
  const float ls = log2_sum(q), lse = log_sum(q, 1.0f);
  float m = q.m, loss = 0.0f;
  counts = t != ignore_index;
  if (counts) {
    if (t < 0 || t >= vocab) loss = m = qnan();
    else if (m != ninf()) loss = fmaf(ls, kLn2, m - logit(t)) + (z_loss == 0.0f ? 0.0f : z_loss * lse * lse);
  }
  row_loss[row] = loss;
  stats[row] = m;
  stats[rows + row] = ls;
  return loss;
}

// R rows a block, THREADS / R lanes each: joins the tiles' maxima and sums, four of a lane's at a time.  A block also sums
// its rows' losses: closes the reduced loss if it has all rows, leaves its sums in `pairs` otherwise.  3 to 11 us, latency.
template <int R, int THREADS>
__global__ __launch_bounds__(THREADS) void k_ce_rows(const float2* __restrict__ partial, int64_t rows_padded, int tiles,
                                                      const float* __restrict__ target_logit,
                                                      const int64_t* __restrict__ target, int64_t ignore_index, int64_t vocab,
                                                      float z_loss, int64_t rows, float* __restrict__ row_loss,
                                                      float* __restrict__ stats, int reduction, double* __restrict__ pairs,
                                                      float* __restrict__ loss_out, float* __restrict__ divisor) {
  constexpr int P = THREADS / R;
  __shared__ float2 part[P][R];
  const int r = threadIdx.x % R, g = threadIdx.x / R;
  const int64_t row = (int64_t)blockIdx.x * R + r;
  MaxSum q{ninf(), 0.0f};
  if (row < rows)
    for (int i = g; i < tiles; i += 4 * P) {
      float2 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        p[u] = i + u * P < tiles ? partial[(int64_t)(i + u * P) * rows_padded + row] : make_float2(ninf(), 0.0f);
#pragma unroll
      for (int u = 0; u < 4; ++u) q = join(q, {p[u].x, p[u].y}, kLog2e);
    }
  part[g][r] = make_float2(q.m, q.s);
#pragma unroll
  for (int n = P / 2; n >= 1; n >>= 1) {
    __syncthreads();
    if (g < n) {
      q = join(q, {part[g + n][r].x, part[g + n][r].y}, kLog2e);
      part[g][r] = make_float2(q.m, q.s);
    }
  }
  float loss = 0.0f;
  bool counts = false;
  if (g == 0 && row < rows)
    loss = close_row(q, [&](int64_t) { return target_logit[row]; }, target[row], ignore_index, vocab, z_loss, row, rows, row_loss,
                     stats, counts);
  if (reduction == VSL_REDUCE_NONE) return;
  __shared__ double sum[2][R];
  __syncthreads();
  if (g == 0) {
    sum[0][r] = (double)loss;
    sum[1][r] = counts ? 1.0 : 0.0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0, count = 0.0;
    for (int i = 0; i < R; ++i) {
      total += sum[0][i];
      count += sum[1][i];
    }
    if (gridDim.x == 1) {
      finish_sum(total, count, reduction, loss_out, divisor);
    } else {
      pairs[2 * blockIdx.x] = total;
      pairs[2 * blockIdx.x + 1] = count;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// backward: scales of the rows
// ------------------------------------------------------------------------------------------------------------------
// What the products are multiplied by at the end.  Where every row has the same gradient g, the derivatives are made for
// a gradient of `unit` and this is g / unit.  Where they differ (one per row, or by z_loss) a row's derivatives are made for
// its own gradient over a power of two, its size, which puts the largest of them between unit and 2 unit.  grad_hidden's rows
// are multiplied by their sizes again: nothing of a row, however small its gradient, infinite or NaN, meets another's.  The
// other two gradients add up rows: there the derivatives are scaled to the largest size of all, and this is that size.
struct OutScale {
  const float* g_loss;    // NULL: `given` holds the scale
  const float* divisor;   // NULL: 1
  const float* given;
  const float* rows;      // not NULL: one for every row of the output
  float unit;
  __device__ __forceinline__ float gradient() const {
    if (!divisor) return *g_loss;
    return *divisor == 0.0f ? 0.0f : *g_loss / *divisor;
  }
  __device__ __forceinline__ float get() const { return g_loss ? gradient() / unit : *given; }
};

struct ScaleArgs {
  const float* g_loss;
  const float* divisor;  // NULL: 1
  const float* stats;
  const int64_t* target;
  int64_t ignore_index, rows, rows_padded;
  bool per_row;          // g_loss holds one gradient per row
  float z_loss, unit;
  float* partial;        // maxima of the blocks of k_ce_largest
  int partials;
  float* row_scale;      // [rows_padded]
  float* row_size;       // [rows_padded]
  float* out_scale;      // one float
};
__device__ __forceinline__ float row_gradient(const ScaleArgs& a, int64_t row) {
  if (a.target[row] == a.ignore_index || a.stats[row] == ninf()) return 0.0f;
  const OutScale g{a.g_loss + (a.per_row ? row : 0), a.divisor, nullptr, nullptr, 1.0f};
  return g.gradient();
}
// size of a row's largest derivative, 0 where it has none that is finite
__device__ __forceinline__ float row_largest(const ScaleArgs& a, int64_t row, float g) {
  if (!(fabsf(g) < __uint_as_float(0x7F800000u))) return 0.0f;
  const float slope = fabsf(slope_of(a.z_loss, a.stats[row], a.stats[a.rows + row]));  // NaN in a row of NaN
  return fminf(fabsf(g) * fmaxf(1.0f, slope), __uint_as_float(0x7F7FFFFFu));
}
// (below 2^-100 sizes stay there: a gradient of 2^-149 still keeps its bits, and sizes over unit stay normal numbers)
__device__ __forceinline__ int exponent_of(float x) { return x == 0.0f ? 0 : max(ilogbf(x), -100); }
__device__ __forceinline__ float block_max(float v, float* red) {
  v = group_all<64>(v, MaxF());
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(red[0], red[1]),
                                       __builtin_elementwise_maximum(red[2], red[3]));
}
__global__ __launch_bounds__(kThreads) void k_ce_largest(ScaleArgs a) {
  __shared__ float red[4];
  float m = 0.0f;
  for (int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * kThreads)
    m = fmaxf(m, row_largest(a, r, row_gradient(a, r)));
  m = block_max(m, red);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = m;
}
__global__ __launch_bounds__(kThreads) void k_ce_scale(ScaleArgs a) {
  __shared__ float red[4];
  const int all = exponent_of(block_max((int)threadIdx.x < a.partials ? a.partial[threadIdx.x] : 0.0f, red));
  const int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (r < a.rows_padded) {
    const float g = r < a.rows ? row_gradient(a, r) : 0.0f;
    const float largest = r < a.rows ? row_largest(a, r, g) : 0.0f;
    const int own = largest == 0.0f ? all : exponent_of(largest);
    a.row_scale[r] = ldexpf(g, -own) * a.unit;
    a.row_size[r] = ldexpf(1.0f, own) / a.unit;
  }
  if (r == 0) *a.out_scale = ldexpf(1.0f, all) / a.unit;
}

// ------------------------------------------------------------------------------------------------------------------
// layouts
// ------------------------------------------------------------------------------------------------------------------
// Everything that has to be laid out for the products goes in one launch, as jobs with a run of blocks each:
//   copy       out [rows][planes][width] = in [rows, cols], zeros behind
//   transpose  out [cols][planes][width] = in^T, zeros behind; a row that cannot contribute (its target is ignored, no
//              class of it is left, its scale is 0, or, of the weight, its bias is -infinity) reads as zeros, so that a NaN
//              in it does not meet the zero of its derivative
struct Contributes {
  const int64_t* target;
  const float* stats;
  const float* scale;
  const void* bias;
  int64_t ignore_index;
  template <typename T>
  __device__ __forceinline__ bool row(int64_t r) const {
    bool on = true;
    if (target) on = (int)(target[r] != ignore_index) & (int)(stats[r] != ninf());
    if (scale) on &= scale[r] != 0.0f;
    if (bias) on &= (float)((const T*)bias)[r] != ninf();
    return on;
  }
};
struct LayoutJob {
  const void* in;
  void* out;
  int64_t stride, rows, width;  // of in, of in, of out
  int cols;
  bool transpose;
  Contributes with;
  int64_t blocks;
};
struct LayoutJobs {
  LayoutJob job[4];
};

// A float's three planes.  The first is cut off instead of rounded where rounding would leave bfloat16's range.
struct Planes {
  u32x4 h, m, l;
};
__device__ __forceinline__ Planes planes_of(const float (&v)[8]) {
  bf16x8 h, m, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x = v[e];
    h[e] = (__bf16)x;
    if (fabsf((float)h[e]) == __uint_as_float(0x7F800000u)) h[e] = (__bf16)__uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    x -= (float)h[e];
    m[e] = (__bf16)x;
    x -= (float)m[e];
    l[e] = (__bf16)x;
  }
  return {__builtin_bit_cast(u32x4, h), __builtin_bit_cast(u32x4, m), __builtin_bit_cast(u32x4, l)};
}
// eight floats of a row, zeros behind the last column
__device__ __forceinline__ void load8(const float* p, int c, int cols, float (&v)[8]) {
  if (c + 8 <= cols) {
    const u32x4 a = load16(p + c), b = load16(p + c + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = __uint_as_float(a[e]);
      v[4 + e] = __uint_as_float(b[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? p[c + e] : 0.0f;
  }
}
template <typename O>
__device__ __forceinline__ void store_planes(O* out, int64_t width, const Planes& q) {
  *(u32x4*)out = q.h;
  *(u32x4*)(out + width) = q.m;
  *(u32x4*)(out + 2 * width) = q.l;
}

template <typename T, bool SPLIT>
__device__ __forceinline__ void copy_job(const LayoutJob& j, int64_t block) {
  constexpr int E = SPLIT ? 8 : Kind<T>::E;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (int64_t r = block * 4 + y; r < j.rows; r += j.blocks * 4) {
    const T* p = (const T*)j.in + r * j.stride;
    for (int64_t c = x * E; c < j.width; c += 64 * E) {
      if constexpr (SPLIT) {
        float v[8];
        load8(p, (int)c, j.cols, v);
        store_planes((__bf16*)j.out + r * 3 * j.width + c, j.width, planes_of(v));
      } else {
        *(u32x4*)((T*)j.out + r * j.width + c) = load_columns(p, (int)c, j.cols);
      }
    }
  }
}

template <typename T, bool SPLIT>
__device__ __forceinline__ void transpose_job(const LayoutJob& j, int64_t block, char* lds) {
  const int64_t tiles_c = (j.cols + 63) / 64;
  const int64_t r0 = block / tiles_c * 64;
  const int c0 = (int)(block % tiles_c) * 64;
  const T* in = (const T*)j.in;
  if constexpr (sizeof(T) == 2) {
    // A thread takes eight columns of two rows and leaves eight words of two rows each in the columns' lines; a line is
    // 32 words, turned by four words per group of eight columns so that the groups' words meet in different banks.
    unsigned* tile = (unsigned*)lds;
    {
      const int g = threadIdx.x & 7, rp = threadIdx.x >> 3, c = c0 + 8 * g;
      const int64_t r = r0 + 2 * rp;
      u32x4 x{0u, 0u, 0u, 0u}, y = x;
      if (c < j.cols && r < j.rows && j.with.row<T>(r)) x = load_columns(in + r * j.stride, c, j.cols);
      if (c < j.cols && r + 1 < j.rows && j.with.row<T>(r + 1)) y = load_columns(in + (r + 1) * j.stride, c, j.cols);
      unsigned* t = tile + 8 * g * 32 + ((rp + 4 * g) & 31);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[(2 * i) * 32] = (x[i] & 0xFFFFu) | y[i] << 16;
        t[(2 * i + 1) * 32] = x[i] >> 16 | (y[i] & 0xFFFF0000u);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = i * kThreads + threadIdx.x, c = at >> 3, piece = at & 7;
      if (c0 + c < j.cols)
        *(u32x4*)((T*)j.out + (int64_t)(c0 + c) * j.width + r0 + 8 * piece) =
            *(const u32x4*)(tile + c * 32 + ((4 * piece + 4 * (c >> 3)) & 31));
    }
  } else {
    float(*tile)[65] = (float(*)[65])lds;
    const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
    float v[16];
    bool on[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // clamped into the matrix, so that all reads go out together
      const int64_t r = min(r0 + y + 4 * i, j.rows - 1);
      on[i] = j.with.row<T>(r);
      v[i] = in[r * j.stride + min(c0 + x, j.cols - 1)];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) tile[y + 4 * i][x] = on[i] && c0 + x < j.cols && r0 + y + 4 * i < j.rows ? v[i] : 0.0f;
    __syncthreads();
    if constexpr (SPLIT) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = i * kThreads + threadIdx.x, c = at >> 3, piece = at & 7;
        if (c0 + c >= j.cols) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[8 * piece + e][c];
        store_planes((__bf16*)j.out + (int64_t)(c0 + c) * 3 * j.width + r0 + 8 * piece, j.width, planes_of(v));
      }
    } else {
      for (int i = y; i < 64; i += 4)
        if (c0 + i < j.cols) ((T*)j.out)[(int64_t)(c0 + i) * j.width + r0 + x] = tile[x][i];
    }
  }
}

// 16384 x 4096 bfloat16 transposed: 49 us, 5.5 TB/s read and written; planes of 1536 x 512 and 10007 x 512 float32, as they lie
// and transposed: 20 us.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(kThreads) void k_layout(LayoutJobs jobs) {
  __shared__ __attribute__((aligned(16))) char lds[64 * 65 * 4];
  int64_t block = blockIdx.x;
  int n = 0;
  while (block >= jobs.job[n].blocks) block -= jobs.job[n++].blocks;  // the grid is the sum of the jobs' blocks
  const LayoutJob& j = jobs.job[n];
  if (j.transpose) transpose_job<T, SPLIT>(j, block, lds);
  else copy_job<T, SPLIT>(j, block);
}

// ------------------------------------------------------------------------------------------------------------------
// the two gradient products
// ------------------------------------------------------------------------------------------------------------------
struct GradArgs {
  Operands op;             // A: [M features, K], B: [N rows or classes, K]
  int splits;              // of K
  bool add;                // to what `sum` holds
  bool whole;              // four features in a row of `sum` are one aligned store
  float* sum;              // [splits][N][M], or NULL: straight to `out`
  void* out;               // [N][M] of the operands' type
  OutScale scale;
};

// one or both products of a piece: the first job's blocks, then the second's
struct GradJobs {
  GradArgs job[2];
  unsigned first;  // blocks of the first
};

// A tile straight to `out`.  A lane holds four features of 32 rows each: stored from there, a row's line is written in
// eight or sixteen pieces by as many stores.  So the tile goes through LDS first, whole rows leave it, 16 bytes a lane, at
// any address.  Pieces of a row are turned by the row, so that neither side's 16 lanes meet in a bank.  A float32 tile that
// is larger than the LDS goes in two halves of its features.
template <typename T, typename S>
__device__ __forceinline__ void store_tile(const GradArgs& a, int m0, int n0, const Tile<S>& t, char* lds) {
  constexpr int kHalves = S::BM * S::BN * (int)sizeof(T) > S::kLds ? 2 : 1, kWide = S::BM / kHalves;
  constexpr int E = Kind<T>::E, kPieces = kWide / E;  // of a row
  static_assert(kWide * S::BN * (int)sizeof(T) <= S::kLds && kPieces >= 16 && S::WM % kHalves == 0, "tile through LDS");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  float scale[S::JN];
  if (a.scale.rows) {
#pragma unroll
    for (int j = 0; j < S::JN; ++j) scale[j] = a.scale.rows[min(n0 + (wn * S::JN + j) * 32 + (lane & 31), a.op.N - 1)];
  } else {
    scale[0] = a.scale.get();
#pragma unroll
    for (int j = 1; j < S::JN; ++j) scale[j] = scale[0];
  }
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    if (h) __syncthreads();
    if (wm / (S::WM / kHalves) == h) {
#pragma unroll
      for (int j = 0; j < S::JN; ++j)
#pragma unroll
        for (int i = 0; i < S::IM; ++i)
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const int n = (wn * S::JN + j) * 32 + (lane & 31);
            const int m = (wm * S::IM + i) * 32 - h * kWide + 8 * r4 + 4 * (lane >> 5);
            float g[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = scale[j] * t.acc[i][j][4 * r4 + e];
            char* p = lds + (n * kPieces + ((m / E) ^ (n & 15))) * 16;
            if constexpr (sizeof(T) == 4) *(f32x4*)p = f32x4{g[0], g[1], g[2], g[3]};
            else *(uint2*)(p + 8 * (lane >> 5)) = pack4<T>(g);
          }
    }
    __syncthreads();
    for (int at = threadIdx.x; at < S::BN * kPieces; at += S::kThreads) {
      const int n = at / kPieces, piece = at % kPieces, m = m0 + h * kWide + piece * E;
      if (n0 + n >= a.op.N || m >= a.op.M) continue;
      const u32x4 v = *(const u32x4*)(lds + (n * kPieces + (piece ^ (n & 15))) * 16);
      T* out = (T*)a.out + (int64_t)(n0 + n) * a.op.M + m;
      if (m + E <= a.op.M) {
        store16(out, v);
      } else {
        float x[E];
        unpack(v, x, (const T*)nullptr);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (m + e < a.op.M) out[e] = (T)x[e];
      }
    }
  }
}

// 8192 x 131072 x 4096 bfloat16, both products of a piece: 1.757 ms, 1252 TFLOP/s, bound as k_ce_logits is.
template <typename T, typename S, bool SPLIT, int FORM>
__global__ __launch_bounds__(S::kThreads) void k_ce_grad(GradJobs jobs) {
  const int which = blockIdx.x >= jobs.first ? 1 : 0;
  const GradArgs& a = jobs.job[which];
  const int block = blockIdx.x - (which ? jobs.first : 0u);
  __shared__ __attribute__((aligned(16))) char lds[S::kLds];
  const int tm_count = (a.op.M + S::BM - 1) / S::BM, tn_count = (a.op.N + S::BN - 1) / S::BN;
  const int tiles = tm_count * tn_count, split = block / tiles;
  int tm, tn;
  tile_of(block % tiles, tm_count, tn_count, tm, tn);
  const int steps = (SPLIT ? kPairs : 1) * a.op.kblocks, per = (steps + a.splits - 1) / a.splits;
  const int k0 = min(split * per, steps), k1 = min(k0 + per, steps);
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  Tile<S> t;
  tile_product<std::conditional_t<SPLIT, __bf16, T>, S, SPLIT, FORM>(a.op, m0, n0, k0, k1, lds, t);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  if (!a.sum) return store_tile<T, S>(a, m0, n0, t, lds);
#pragma unroll
  for (int j = 0; j < S::JN; ++j) {
    const int row = n0 + (wn * S::JN + j) * 32 + (lane & 31);
    if (row >= a.op.N) continue;
    float* sum = a.sum + (int64_t)split * a.op.M * a.op.N + (int64_t)row * a.op.M;
#pragma unroll
    for (int i = 0; i < S::IM; ++i)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int m = m0 + (wm * S::IM + i) * 32 + 8 * r4 + 4 * (lane >> 5);
        if (a.whole && m < a.op.M) {
          f32x4* p = (f32x4*)(sum + m);
          f32x4 v{t.acc[i][j][4 * r4], t.acc[i][j][4 * r4 + 1], t.acc[i][j][4 * r4 + 2], t.acc[i][j][4 * r4 + 3]};
          if (a.add) v += *p;
          *p = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (m + e < a.op.M) sum[m + e] = a.add ? sum[m + e] + t.acc[i][j][4 * r4 + e] : t.acc[i][j][4 * r4 + e];
        }
      }
  }
}

// out = scale * the sum of the splits, in their order: four elements a thread; many splits are dealt to the four waves; up to
// three sums in one launch.  8192 x 4096 float32 to bfloat16: 49 us, 4.1 TB/s.
constexpr int kDealtSplits = 8;  // at least
struct FinishJob {
  const float* sum;
  void* out;
  int splits;
  int64_t n;
  int64_t blocks;
  const float* row_scale;  // ROWS: of rows of `width` elements, or NULL: jobs' scale
  int64_t width;
};
struct FinishJobs {
  FinishJob job[3];
  OutScale scale;
};
template <typename T, bool ROWS>
__global__ __launch_bounds__(kThreads) void k_ce_finish(FinishJobs jobs) {
  __shared__ f32x4 part[3][64];
  int64_t block = blockIdx.x;
  int which = 0;
  while (block >= jobs.job[which].blocks) block -= jobs.job[which++].blocks;  // the grid is the sum of the jobs' blocks
  const FinishJob& j = jobs.job[which];
  const float scale = jobs.scale.get();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto sum = [&](int64_t i, int s0, int s1) {
    f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
    if (i + 4 <= j.n) {
#pragma unroll 8
      for (int s = s0; s < s1; ++s) v += __builtin_bit_cast(f32x4, load16(j.sum + s * j.n + i));
    } else if (i < j.n) {
      for (int s = s0; s < s1; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < j.n) v[e] += j.sum[s * j.n + i + e];
    }
    return v;
  };
  auto store = [&](int64_t i, const f32x4& v) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < j.n) ((T*)j.out)[i + e] = (T)((ROWS && j.row_scale ? j.row_scale[(i + e) / j.width] : scale) * v[e]);
  };
  if (j.splits < kDealtSplits) {
    for (int64_t i = (block * kThreads + threadIdx.x) * 4; i < j.n; i += j.blocks * kThreads * 4) store(i, sum(i, 0, j.splits));
    return;
  }
  const int per = (j.splits + 3) / 4, s0 = min(j.splits, wave * per), s1 = min(j.splits, s0 + per);
  for (int64_t i0 = block * 256; i0 < j.n; i0 += j.blocks * 256) {
    const int64_t i = i0 + 4 * lane;
    f32x4 v = sum(i, s0, s1);
    __syncthreads();
    if (wave) part[wave - 1][lane] = v;
    __syncthreads();
    if (wave) continue;
#pragma unroll
    for (int w = 0; w < 3; ++w) v += part[w][lane];
    store(i, v);
  }
}

// grad_bias: sums of the rows of d^T, the values that grad_weight is made of; L lanes per class and part of its row
template <typename T, bool SPLIT, int L>
__global__ __launch_bounds__(kThreads) void k_ce_bias(const void* __restrict__ delta_t, int64_t ldt, int64_t rows_padded,
                                                      int64_t rows, int classes, int parts, float* __restrict__ sum,
                                                      OutScale out_scale, T* __restrict__ out) {
  typedef std::conditional_t<SPLIT, __bf16, T> O;
  __shared__ float red[4];
  const int item = blockIdx.x * (kThreads / L) + threadIdx.x / L, lane = threadIdx.x % L;
  if (item >= classes * parts) return;  // whole groups of L
  const int c = item % classes, part = item / classes;
  const int64_t vectors = rows / Kind<O>::E, per = (vectors + parts - 1) / parts;
  const int64_t end = min(vectors, (part + 1) * per);
  float s = 0.0f;
  for (int plane = SPLIT ? 2 : 0; plane >= 0; --plane) {
    const O* d = (const O*)delta_t + (int64_t)c * ldt + plane * rows_padded;
    for (int64_t i = part * per + lane; i < end; i += L) {
      float x[Kind<O>::E];
      unpack(load16(d + i * Kind<O>::E), x, (const O*)nullptr);
#pragma unroll
      for (int e = 0; e < Kind<O>::E; ++e) s += x[e];
    }
  }
  if constexpr (L == kThreads) s = block_add<4>(s, red);
  else s = group_all<L>(s, AddF());
  if (lane) return;
  if (sum) sum[(int64_t)part * classes + c] = s;
  else out[c] = (T)(s * out_scale.get());
}

// ------------------------------------------------------------------------------------------------------------------
// Logits in parts of the features: few tiles over many features leave most CUs idle, so the product is cut along them
// like the gradients' and leaves [splits][rows][classes] sums, from which these two take their logits.  12 x 1398 x 1944
// float32 forward: 16 us, whole 69; 459 x 767 x 3722 with gradients: 210 and 503; 200 x 1000 x 4096 bfloat16 forward: 15 and
// 40.  Both kernels are bound by the latency of their reads, which is why these go out 16 at a time.
// ------------------------------------------------------------------------------------------------------------------
struct Parts {
  const float* sum;
  int splits;
  int64_t rows, vocab;
  const void* bias;
  // U logits `apart` elements apart, the first of them `row`, `v`; -infinity where `on` says no
  template <typename T, int U, typename On>
  __device__ __forceinline__ void logits(int64_t row, int64_t v, int64_t rows_apart, int64_t classes_apart, On on,
                                         float (&z)[U]) const {
    const int64_t all = rows * vocab;
    const float* p[U];  // every one is read, so that the reads go out together
#pragma unroll
    for (int u = 0; u < U; ++u) {
      z[u] = 0.0f;
      p[u] = sum + (on(u) ? (row + u * rows_apart) * vocab + v + u * classes_apart : 0);
    }
    int s = 0;
    for (; s + 4 <= splits; s += 4) {
      float x[4][U];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) x[i][u] = p[u][(s + i) * all];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) z[u] += x[i][u];
    }
    for (; s < splits; ++s)
#pragma unroll
      for (int u = 0; u < U; ++u) z[u] += p[u][s * all];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float b = !on(u) ? ninf() : bias ? (float)((const T*)bias)[v + u * classes_apart] : 0.0f;
      z[u] = b == ninf() ? b : z[u] + b;  // a masked class stays masked whatever its weights hold
    }
  }
  template <typename T>
  __device__ __forceinline__ float logit(int64_t row, int64_t v) const {
    float z[1];
    logits<T>(row, v, 0, 0, [](int) { return true; }, z);
    return z[0];
  }
};

// forward: a block per row
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_ce_parts_rows(Parts z, const int64_t* __restrict__ target, int64_t ignore_index,
                                                           float z_loss, float* __restrict__ row_loss,
                                                           float* __restrict__ stats, int reduction,
                                                           double* __restrict__ pairs, float* __restrict__ loss_out,
                                                           float* __restrict__ divisor) {
  __shared__ float red[THREADS / 32];
  const int64_t row = blockIdx.x;
  RunSum run;
  for (int64_t v = threadIdx.x; v < z.vocab; v += 4 * THREADS) {
    float x[4];
    z.logits<T>(row, v, 0, THREADS, [&](int u) { return v + u * THREADS < z.vocab; }, x);
    float m = run.m;
#pragma unroll
    for (int u = 0; u < 4; ++u) m = __builtin_elementwise_maximum(m, x[u]);
    const Exponent ex = run.move(m, kLog2e);
#pragma unroll
    for (int u = 0; u < 4; ++u) run.s += ex(x[u]);
  }
  const MaxSum q = block_join<THREADS / 64>(run.get(), red, kLog2e);
  if (threadIdx.x) return;
  bool counts;
  const float loss = close_row(q, [&](int64_t t) { return z.logit<T>(row, t); }, target[row], ignore_index, z.vocab, z_loss, row,
                               z.rows, row_loss, stats, counts);
  if (reduction == VSL_REDUCE_NONE) return;
  if (gridDim.x == 1) {
    finish_sum((double)loss, counts ? 1.0 : 0.0, reduction, loss_out, divisor);
  } else {
    pairs[2 * row] = (double)loss;
    pairs[2 * row + 1] = counts ? 1.0 : 0.0;
  }
}

// backward: 16 rows x 64 classes a block, written as they are and transposed
constexpr int kPartRows = 16;
template <typename T>
__global__ __launch_bounds__(kThreads) void k_ce_parts_delta(Parts z, LogitArgs a) {
  __shared__ float tile[kPartRows][65];
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int64_t r0 = (int64_t)blockIdx.y * kPartRows, v0 = (int64_t)blockIdx.x * 64, v = v0 + x;
  float logit[4];
  z.logits<T>(r0 + y, v, 4, 0, [&](int u) { return r0 + y + 4 * u < z.rows && v < z.vocab; }, logit);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t row = r0 + y + 4 * u;
    const bool live = row < z.rows;
    const int64_t target = live ? a.target[row] : -1;
    const float top = live ? a.stats[row] : ninf(), ls = live ? a.stats[z.rows + row] : 0.0f;
    const float scale = !live || top == ninf() || target == a.ignore_index ? 0.0f : a.row_scale ? a.row_scale[row] : a.unit;
    float d = 0.0f;
    if (scale != 0.0f) {
      const Exponent ex(top, kLog2e);
      d = scale * slope_of(a.z_loss, top, ls) * ex.factor(ls) * ex(logit[u]);
      if (v == target) d -= scale;
    }
    if (a.delta) ((T*)a.delta)[row * a.ldd + v] = (T)d;
    tile[y + 4 * u][x] = live && a.row_scale ? d * (a.row_size[row] / *a.out_scale) : d;
  }
  if (!a.delta_t) return;
  __syncthreads();
  const int r = threadIdx.x % kPartRows;
#pragma unroll
  for (int c = threadIdx.x / kPartRows; c < 64; c += kThreads / kPartRows) ((T*)a.delta_t)[(v0 + c) * a.ldt + r0 + r] = (T)tile[r][c];
}

// ------------------------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------------------------
int size_of(int type) { return type == VSL_TYPE_F32 ? 4 : 2; }
int64_t round_up(int64_t v, int64_t to) { return ceil_div(v, to) * to; }

int check_ce(const vsl_linear_ce_desc* d) {
  if (!d) return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: descriptor is null");
  if (d->type != VSL_TYPE_F32 && d->type != VSL_TYPE_BF16 && d->type != VSL_TYPE_F16)
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: unknown element type");
  if (d->rows < 0 || d->rows >= (1LL << 28) || d->vocab < 1 || d->vocab >= (1LL << 30) || d->dim < 1 || d->dim >= (1LL << 24))
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: need 0 <= rows < 2^28, 1 <= vocab < 2^30, 1 <= dim < 2^24");
  // a launch counts its threads in 32 bits: tiles of 128 x 64 by 256 threads, blocks of 64 x 64 laid out by 256
  if (round_up(d->rows, 256) * round_up(d->vocab, 256) >= (1LL << 37) ||
      round_up(d->rows, 256) * round_up(d->dim, 64) >= (1LL << 34) || round_up(d->vocab, 256) * round_up(d->dim, 64) >= (1LL << 34))
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: need rows * vocab < 2^37, rows * dim < 2^34 and vocab * dim < 2^34");
  if (d->hidden_stride < d->dim || d->weight_stride < d->dim || d->hidden_stride >= (1LL << 40) || d->weight_stride >= (1LL << 40))
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: row strides must be at least dim");
  if (d->reduction < VSL_REDUCE_NONE || d->reduction > VSL_REDUCE_MEAN)
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: unknown reduction");
  if (!(d->z_loss >= 0.0f) || d->z_loss > 1e30f) return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: z_loss must be finite and not negative");
  if (!d->weight || (d->rows > 0 && (!d->hidden || !d->target))) return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: NULL tensor");
  const int s = size_of(d->type);
  if ((uintptr_t)d->hidden % s || (uintptr_t)d->weight % s || (uintptr_t)d->bias % s)
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: misaligned tensor");
  return VSL_OK;
}

// An operand goes to the main loop as it is when its rows are whole 16-byte pieces at 16-byte addresses.
bool ready(const void* p, int64_t stride, int64_t dim, int type) {
  const int s = size_of(type);
  return (uintptr_t)p % 16 == 0 && stride * s % 16 == 0 && dim * s % 16 == 0;
}

struct Arena {
  char* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base ? base + used : nullptr;
    used += up256(bytes);
    return p;
  }
};

struct Plan {
  int shape, splits;  // of the tiles of a product, and of its K
  double time;        // estimated, microseconds
};
enum { kLarge, kSmall, kNarrow, kThin };
struct ShapeInfo {
  int bm, bn, slots;             // tile, and how many of it the 256 CUs hold at once
  float step16, step32, around;  // microseconds of a step of K with all slots taken (16-bit types, float32), and of a tile's
                                 // beginning and end
};
// Measured on products of 2048..8192 rows (large: 1240 TFLOP/s in bfloat16, small: 850; float32: 105).
constexpr ShapeInfo kShapes[] = {{Large::BM, Large::BN, 256, 1.7f, 0.0f, 4.0f},
                                 {Small::BM, Small::BN, 512, 1.3f, 5.0f, 2.5f},
                                 {Narrow::BM, Narrow::BN, 768, 1.1f, 4.0f, 2.0f},
                                 {Thin::BM, Thin::BN, 1024, 1.0f, 3.0f, 1.5f}};
// A step through registers against one straight to LDS, its loads off their alignment.  7 x 96190 x 3653 bfloat16 forward
// takes 161 us through registers and 420 copied first; 6439 x 736 x 2647 float16 with gradients 297 and 271.
constexpr double kStaged = 1.5;
// Shape of the tiles of a product M x N over `blocks` steps of K, and into how many parts K is cut: the least of the waves
// of tiles times their length, plus the traffic of the partial sums.  float32 leaves out the large tile: its epilogue
// does not fit the registers, and its matrix instructions are eight times slower, so that its loads never bind.
Plan plan_of(int64_t M, int64_t N, int64_t blocks, int type, bool may_split, bool staged = false, int only = -1) {
  Plan best{kSmall, 1, 1e300};
  // the thin tile: float32 is bound by its multiplications, of which up to three of it waste fewer (67 x 113867 x 1013
  // forward: 245 us, with two of the narrow one 270); 16-bit types by reading A
  const int last = N <= (type == VSL_TYPE_F32 ? 3 : 1) * Thin::BN ? kThin : kNarrow;
  for (int shape = type == VSL_TYPE_F32 || staged ? kSmall : kLarge; shape <= last; ++shape) {
    if (only >= 0 && shape != only) continue;
    const ShapeInfo& h = kShapes[shape];
    const double tiles = (double)(ceil_div(M, h.bm) * ceil_div(N, h.bn));
    const double step = (type == VSL_TYPE_F32 ? h.step32 : h.step16) * (staged ? kStaged : 1.0);
    for (int s = 1; s <= 256 && (s == 1 || (may_split && blocks / s >= 4)); s = s < 16 ? s + 1 : s + s / 4) {
      // a CU that holds fewer tiles than it could runs each of them faster, though not in proportion
      const double full = (double)(int64_t)(tiles * s / h.slots), rest = tiles * s - full * h.slots;
      const double per_cu = h.slots / 256.0, held = (double)(int64_t)((rest + 255) / 256);
      double t = (full + (rest > 0 ? 0.1 + 0.9 * held / per_cu : 0.0)) * ((double)ceil_div(blocks, s) * step + h.around);
      if (s > 1) t += 4.0 + (double)s * (double)M * (double)N * 8.0 / 4e6;
      if (t < best.time) best = {shape, s, t};
    }
  }
  return best;
}
int64_t blocks_of(int64_t K, int type) { return ceil_div(K * size_of(type), kBlockBytes); }


// How the operands of the products lie: elements of `size` bytes, `planes` of them a value, BK elements a step.
struct Layout {
  bool split;          // float32 by planes of bfloat16
  int type, size, planes;
  int64_t rows_padded, dim_padded;
  bool copy_hidden, copy_weight;
  bool staged;         // the logits' operands go through registers
  int tail;            // Operands::tail of the logits' products
  Plan logits;         // of the logits of all classes; several splits: in parts
  int64_t steps(int64_t K) const { return (split ? kPairs : 1) * blocks_of(K, type); }
};
constexpr int64_t kMostParts = 1LL << 23;  // padded logits whose product may be cut: with more there are tiles enough
Layout layout_of(const vsl_linear_ce_desc* d) {
  Layout l{};
  l.rows_padded = round_up(d->rows, kPad);
  // Logits in parts cost a pass over the sums, forward and backward (5 us, 3 more to launch
  // it, and 0.5 for every turn of its block along a row).
  auto plan_logits = [&](int type, int64_t steps, bool parts, bool staged) {
    const Plan whole = plan_of(d->vocab, d->rows, steps, type, false, staged);
    if (!parts || l.rows_padded * round_up(d->vocab, kPad) > kMostParts) return whole;
    Plan cut = plan_of(d->vocab, d->rows, steps, type, true, staged);
    cut.time += 8.0 + 0.5 * (double)ceil_div(d->vocab, 4096);
    return cut.splits > 1 && cut.time < whole.time ? cut : whole;
  };
  l.logits = plan_logits(d->type, blocks_of(d->dim, d->type), true, false);
  l.copy_hidden = !ready(d->hidden, d->hidden_stride, d->dim, d->type);
  l.copy_weight = !ready(d->weight, d->weight_stride, d->dim, d->type);
  if (l.copy_hidden || l.copy_weight) {
    // Rows that the main loop cannot take as they are: copied (read and written), or through registers, without the large
    // tile.
    const int64_t elements = (l.copy_hidden ? d->rows : 0) + (l.copy_weight ? d->vocab : 0);
    l.logits.time += 3.0 + (double)(elements * d->dim * size_of(d->type)) * 2.0 / 4e6;
    const Plan staged = plan_logits(d->type, blocks_of(d->dim, d->type), true, true);
    l.staged = staged.time < l.logits.time;
    if (l.staged) l.logits = staged;
  }
  if (d->type == VSL_TYPE_F32) {
    // the planes are worth writing (10 bytes a value) where they save more on the logits than that
    const Plan planes = plan_logits(VSL_TYPE_BF16, kPairs * blocks_of(d->dim, VSL_TYPE_BF16), false, false);
    l.split = planes.time + 10.0 + (double)(d->rows + d->vocab) * (double)d->dim * 10.0 / 4e6 < l.logits.time;
    if (l.split) l.logits = planes;
  }
  if (l.split) l.staged = false;
  l.type = l.split ? VSL_TYPE_BF16 : d->type;
  l.size = size_of(l.type);
  l.planes = l.split ? 3 : 1;
  l.dim_padded = round_up(d->dim, kBlockBytes / l.size);
  l.copy_hidden = l.split || (l.copy_hidden && !l.staged);
  l.copy_weight = l.split || (l.copy_weight && !l.staged);
  // a copy is padded with zeros up to the block's end; beside an operand that is read in place only its pieces count
  l.tail = l.copy_hidden && l.copy_weight ? 8 : (int)((d->dim * l.size % kBlockBytes + 15) / 16);
  if (l.tail == 0) l.tail = 8;
  return l;
}

// Pieces of the vocabulary: at most this many derivatives (256 MiB in 16 bits, twice), and at most a GiB of a weight that is laid
// out (300 x 131072 x 4096 bfloat16: one piece 2.48 ms, two 2.55, four 2.58).  Smaller pieces would stay in the last-level cache,
// but every piece reads and writes grad_hidden's sums: at 8192 x 131072 x 4096 in bfloat16 2^26, 2^27 and 2^28 derivatives take
// 29.6, 29.3 and 29.3 ms.  Pieces are equal but for a tile: a short last one costs nearly as much as a whole one.
constexpr int64_t kPieceElements = 1LL << 27, kPieceWeight = 1LL << 30;
static_assert(kMostParts <= kPieceElements && kMostParts / kPad / kPartRows < 65536, "logits in parts are one piece, their rows one grid");
struct Pieces {
  int64_t piece, pieces;  // classes of a piece, the last may have fewer
};
// derivatives: of a class; laid_out: bytes a class takes in a layout, 0 without any; tile: what a single piece is padded to
Pieces pieces_of(const vsl_linear_ce_desc* d, int64_t derivatives, int64_t laid_out, int64_t tile) {
  int64_t most = d->vocab;
  if (derivatives > 0) most = std::min(most, std::max(kPieceElements / derivatives / kPad, (int64_t)1) * kPad);
  if (laid_out > 0) most = std::min(most, std::max(kPieceWeight / laid_out / kPad, (int64_t)1) * kPad);
  const int64_t n = ceil_div(d->vocab, most), piece = round_up(ceil_div(d->vocab, n), n == 1 ? tile : kPad);
  return {piece, ceil_div(d->vocab, piece)};
}

struct Forward {
  Layout l;
  Pieces p;
  void *hidden, *weight;
  float2* partial;
  float* target_logit;
  float* parts;
  double* pairs;
  size_t total;
};
Forward forward_workspace(const vsl_linear_ce_desc* d, void* base) {
  Forward f{};
  f.l = layout_of(d);
  const Layout& l = f.l;
  const int s = l.size * l.planes;
  Arena a{(char*)base};
  f.p = pieces_of(d, 0, l.copy_weight && l.logits.splits == 1 ? l.dim_padded * s : 0, kPad);
  f.hidden = l.copy_hidden ? a.take((size_t)d->rows * l.dim_padded * s) : nullptr;
  f.weight = l.copy_weight ? a.take((size_t)(f.p.pieces == 1 ? d->vocab : f.p.piece) * l.dim_padded * s) : nullptr;
  if (l.logits.splits > 1) {
    f.parts = (float*)a.take((size_t)l.logits.splits * d->rows * d->vocab * 4);
    f.pairs = (double*)a.take((size_t)d->rows * 2 * sizeof(double));
    f.total = a.used;
    return f;
  }
  f.partial = (float2*)a.take((size_t)ceil_div(d->vocab, Small::BM) * l.rows_padded * sizeof(float2));
  f.target_logit = (float*)a.take((size_t)d->rows * 4);
  f.pairs = (double*)a.take((size_t)ceil_div(d->rows, d->rows <= 2048 ? 4 : 16) * 2 * sizeof(double));
  f.total = a.used;
  return f;
}

constexpr int64_t kBiasBlocks = 1024;

// grad_hidden of few rows takes a large weight as it lies: transposing it first reads and writes it once more.
// 5 x 60478 x 1627 float32 with gradients takes 481 us, transposed 746; 57 x 90227 x 1024 float16 263 and 295; above 128 rows
// the gathers bind (346 x 30813 x 1495 float16: 552 and 394), below 16 MB the further launch (19 x 56371 x 54 bfloat16: 104
// and 90).
constexpr int64_t kColumnsRows = 128, kColumnsBytes = 16 << 20;

struct Backward {
  Layout l;
  bool columns;
  int64_t piece, pieces;
  Plan plan_h, plan_w;
  void *hidden, *weight, *hidden_t, *weight_t, *delta, *delta_t;
  float *sum_h, *sum_w, *sum_b, *row_scale, *row_size, *out_scale, *largest, *parts;
  size_t total;
};
Backward backward_workspace(const vsl_linear_ce_desc* d, uint32_t mask, void* base) {
  Backward b{};
  b.l = layout_of(d);
  const int s = b.l.size * b.l.planes;
  const bool gh = mask & 1, gw = mask & 2, gb = mask & 4;
  // dim: a piece that runs over the end of a row has to end in the next one (kStagedColumns)
  const bool columns = !b.l.split && d->rows <= kColumnsRows && d->dim >= 8 && d->vocab * d->dim * size_of(d->type) >= kColumnsBytes;
  b.columns = gh && columns;
  // the same pieces whichever gradients are asked for, so that each has the same bits alone; whole where the logits come in parts
  const bool parts = b.l.logits.splits > 1;
  const int64_t tile = parts ? 64 : kShapes[b.l.logits.shape].bm;
  const int64_t laid_out = columns && !b.l.copy_weight ? 0 : b.l.dim_padded * s;
  const Pieces p = parts ? Pieces{round_up(d->vocab, tile), 1} : pieces_of(d, b.l.rows_padded, laid_out, tile);
  b.piece = p.piece;
  b.pieces = p.pieces;
  Arena a{(char*)base};
  b.hidden = b.l.copy_hidden ? a.take((size_t)d->rows * b.l.dim_padded * s) : nullptr;
  b.weight = b.l.copy_weight ? a.take((size_t)(b.pieces == 1 ? d->vocab : b.piece) * b.l.dim_padded * s) : nullptr;
  b.hidden_t = gw ? a.take((size_t)d->dim * b.l.rows_padded * s) : nullptr;
  b.weight_t = gh && !b.columns ? a.take((size_t)d->dim * b.piece * s) : nullptr;
  b.delta = gh ? a.take((size_t)b.l.rows_padded * b.piece * s) : nullptr;
  b.delta_t = gw || gb ? a.take((size_t)b.l.rows_padded * b.piece * s) : nullptr;
  b.plan_h = plan_of(d->dim, d->rows, b.l.steps(b.piece), b.l.type, true, columns);
  b.plan_w = plan_of(d->dim, d->vocab < b.piece ? d->vocab : b.piece, b.l.steps(d->rows), b.l.type, true);
  if (!columns) {  // tiles of one shape go in one launch, which is worth 4 us; the same where one gradient is asked for alone
    for (int shape = kLarge; shape <= kNarrow && b.plan_h.shape != b.plan_w.shape; ++shape) {
      const Plan h = plan_of(d->dim, d->rows, b.l.steps(b.piece), b.l.type, true, false, shape);
      const Plan w = plan_of(d->dim, d->vocab < b.piece ? d->vocab : b.piece, b.l.steps(d->rows), b.l.type, true, false, shape);
      if (h.time + w.time < b.plan_h.time + b.plan_w.time + 4.0) b.plan_h = h, b.plan_w = w;
    }
  }
  b.sum_h = gh && (b.pieces > 1 || b.plan_h.splits > 1) ? (float*)a.take((size_t)b.plan_h.splits * d->rows * d->dim * 4) : nullptr;
  b.sum_w = gw && b.plan_w.splits > 1 ? (float*)a.take((size_t)b.plan_w.splits * b.piece * d->dim * 4) : nullptr;
  b.sum_b = gb && d->rows >= 8192 && d->vocab <= kBiasBlocks / 2 ? (float*)a.take(kBiasBlocks * 4) : nullptr;
  b.row_scale = (float*)a.take((size_t)b.l.rows_padded * 4);
  b.row_size = (float*)a.take((size_t)b.l.rows_padded * 4);
  b.out_scale = (float*)a.take(4);
  b.largest = (float*)a.take(256 * 4);
  b.parts = b.l.logits.splits > 1 ? (float*)a.take((size_t)b.l.logits.splits * d->rows * d->vocab * 4) : nullptr;
  b.total = a.used;
  return b;
}

dim3 linear_grid(int64_t n) {
  const int64_t b = ceil_div(n, kThreads);
  return dim3((unsigned)(b < 1 ? 1 : (b > 65536 ? 65536 : b)));
}

struct LayoutLaunch {
  LayoutJobs jobs{};
  int n = 0;
  int64_t blocks = 0;
  void add(const LayoutJob& j) {
    jobs.job[n++] = j;
    blocks += j.blocks;
  }
  void copy(const void* in, int64_t stride, int64_t rows, int64_t cols, int64_t width, void* out) {
    const int64_t b = ceil_div(rows, 4);
    add({in, out, stride, rows, width, (int)cols, false, {}, b < 16384 ? b : 16384});
  }
  // covers the first `padded` columns of out's rows (a multiple of 64), zeros behind `rows`
  void transpose(const void* in, int64_t stride, int64_t rows, int64_t cols, int64_t width, int64_t padded, const Contributes& with,
                 void* out) {
    add({in, out, stride, rows, width, (int)cols, true, with, padded / 64 * ceil_div(cols, 64)});
  }
  template <typename T, bool SPLIT>
  void run(hipStream_t s) {
    if (n) hipLaunchKernelGGL((k_layout<T, SPLIT>), dim3((unsigned)blocks), dim3(kThreads), 0, s, jobs);
  }
};
struct FinishLaunch {
  FinishJobs jobs{};
  int n = 0;
  int64_t blocks = 0;
  void add(const float* sum, int splits, int64_t elements, void* out, const float* row_scale = nullptr, int64_t width = 1) {
    const int64_t b = ceil_div(elements, splits < kDealtSplits ? 4 * kThreads : kThreads);
    jobs.job[n++] = {sum, out, splits, elements, b < 65536 ? b : 65536, row_scale, width};
    blocks += jobs.job[n - 1].blocks;
  }
  template <typename T>
  void run(const OutScale& scale, bool rows, hipStream_t s) {
    jobs.scale = scale;
    const auto kernel = rows ? k_ce_finish<T, true> : k_ce_finish<T, false>;
    if (n) hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, s, jobs);
  }
};

template <typename T, typename S, int WHAT, bool SPLIT, int FORM>
int launch_logits_as(const LogitArgs& a, hipStream_t s) {
  const int64_t tm = ceil_div(a.op.M, S::BM), tn = ceil_div(a.op.N, S::BN);
  hipLaunchKernelGGL((k_ce_logits<T, S, WHAT, SPLIT, FORM>), dim3((unsigned)(tm * tn)), dim3(S::kThreads), 0, s, a);
  return (int)tm;
}
// The thin tile: not for derivatives in 16 bits, whose steps of K are 64 rows (run_backward takes the narrow one), nor by planes,
// whose time on it is the direct form's and the layouts' on top.
template <typename T, int WHAT, bool SPLIT>
int launch_logits(const LogitArgs& a, int shape, bool staged, hipStream_t s) {  // returns the rows of tiles
  constexpr bool kHasThin = !SPLIT && (WHAT == kStatistics || sizeof(T) == 4);
  if constexpr (!SPLIT)
    if (staged) {
      if constexpr (kHasThin)
        if (shape == kThin) return launch_logits_as<T, Thin, WHAT, SPLIT, kStagedRows>(a, s);
      if (shape == kNarrow) return launch_logits_as<T, Narrow, WHAT, SPLIT, kStagedRows>(a, s);
      return launch_logits_as<T, Small, WHAT, SPLIT, kStagedRows>(a, s);
    }
  if constexpr (sizeof(T) == 2 || SPLIT)
    if (shape == kLarge) return launch_logits_as<T, Large, WHAT, SPLIT, kDirect>(a, s);
  if constexpr (kHasThin)
    if (shape == kThin) return launch_logits_as<T, Thin, WHAT, SPLIT, kDirect>(a, s);
  if (shape == kNarrow) return launch_logits_as<T, Narrow, WHAT, SPLIT, kDirect>(a, s);
  return launch_logits_as<T, Small, WHAT, SPLIT, kDirect>(a, s);
}
template <typename T, typename S, bool SPLIT, int FORM = kDirect>
void launch_grad_as(const GradArgs* g, int n, hipStream_t s) {
  GradJobs jobs{};
  unsigned blocks = 0;
  for (int i = 0; i < n; ++i) {
    jobs.job[i] = g[i];
    if (i) jobs.first = blocks;
    blocks += (unsigned)(ceil_div(g[i].op.M, S::BM) * ceil_div(g[i].op.N, S::BN) * g[i].splits);
  }
  if (n == 1) jobs.first = blocks;
  hipLaunchKernelGGL((k_ce_grad<T, S, SPLIT, FORM>), dim3(blocks), dim3(S::kThreads), 0, s, jobs);
}
// n products, one after the other in one launch where their tiles have one shape
template <typename T, bool SPLIT>
void launch_grad(GradArgs* g, const int* shape, int n, hipStream_t s) {
  for (int i = 0; i < n; ++i) g[i].whole = g[i].op.M % 4 == 0;
  if (n == 2 && shape[0] != shape[1]) {
    launch_grad<T, SPLIT>(g, shape, 1, s);
    launch_grad<T, SPLIT>(g + 1, shape + 1, 1, s);
    return;
  }
  if (!n) return;
  if constexpr (sizeof(T) == 2 || SPLIT)
    if (shape[0] == kLarge) return launch_grad_as<T, Large, SPLIT>(g, n, s);
  if (shape[0] == kThin) return launch_grad_as<T, Thin, SPLIT>(g, n, s);
  if (shape[0] == kNarrow) return launch_grad_as<T, Narrow, SPLIT>(g, n, s);
  launch_grad_as<T, Small, SPLIT>(g, n, s);
}

template <typename T>
void launch_parts(const Operands& op, const Layout& l, float* parts, hipStream_t s) {
  GradArgs g{};
  g.op = op;
  g.sum = parts;
  g.splits = l.logits.splits;
  g.whole = op.M % 4 == 0;
  if (l.staged && l.logits.shape == kThin) launch_grad_as<T, Thin, false, kStagedRows>(&g, 1, s);
  else if (l.staged && l.logits.shape == kNarrow) launch_grad_as<T, Narrow, false, kStagedRows>(&g, 1, s);
  else if (l.staged) launch_grad_as<T, Small, false, kStagedRows>(&g, 1, s);
  else launch_grad<T, false>(&g, &l.logits.shape, 1, s);
}

template <typename T, bool SPLIT>
void run_forward(const vsl_linear_ce_desc* d, const Forward& f, float* row_loss, float* stats, float* loss,
                 float* divisor, hipStream_t s) {
  typedef std::conditional_t<SPLIT, __bf16, T> O;
  const Layout& l = f.l;
  const O* hidden = (const O*)(l.copy_hidden ? f.hidden : d->hidden);
  int tiles = 0;
  for (int64_t p = 0; p < f.p.pieces; ++p) {
    const int64_t v0 = p * f.p.piece, classes = d->vocab - v0 < f.p.piece ? d->vocab - v0 : f.p.piece;
    const T* given = (const T*)d->weight + v0 * d->weight_stride;
    LayoutLaunch lay;
    if (l.copy_hidden && p == 0) lay.copy(d->hidden, d->hidden_stride, d->rows, d->dim, l.dim_padded, f.hidden);
    if (l.copy_weight) lay.copy(given, d->weight_stride, classes, d->dim, l.dim_padded, f.weight);
    lay.run<T, SPLIT>(s);
    LogitArgs a{};
    a.op = {l.copy_weight ? f.weight : (const void*)given, hidden, l.copy_weight ? l.planes * l.dim_padded : d->weight_stride,
            l.copy_hidden ? l.planes * l.dim_padded : d->hidden_stride, (int)classes, (int)d->rows,
            (int)(l.dim_padded / Kind<O>::BK), l.dim_padded, l.dim_padded, l.tail, (int)d->dim};
    if constexpr (SPLIT) a.given_a = given, a.given_b = (const T*)d->hidden;
    a.given_lda = d->weight_stride;
    a.given_ldb = d->hidden_stride;
    a.bias = d->bias;
    a.target = d->target;
    a.ignore_index = d->ignore_index;
    a.class0 = v0;
    a.rows_padded = l.rows_padded;
    if constexpr (!SPLIT)
      if (f.parts) {
        launch_parts<T>(a.op, l, f.parts, s);
        auto rows = [&](auto kernel, int threads) {
          hipLaunchKernelGGL(kernel, dim3((unsigned)d->rows), dim3(threads), 0, s,
                             Parts{f.parts, l.logits.splits, d->rows, d->vocab, d->bias}, d->target, d->ignore_index, d->z_loss,
                             row_loss, stats, d->reduction, f.pairs, loss, divisor);
        };
        if (d->vocab > 2048) rows(k_ce_parts_rows<T, 1024>, 1024);  // 10544 classes of two rows: 8.9 us, with 256 threads 17.6
        else rows(k_ce_parts_rows<T, kThreads>, kThreads);
        if (d->reduction != VSL_REDUCE_NONE && d->rows > 1) launch_sum_pairs(f.pairs, d->rows, d->reduction, loss, divisor, s);
        return;
      }
    a.partial = f.partial + tiles * l.rows_padded;
    a.target_logit = f.target_logit;
    tiles += launch_logits<T, kStatistics, SPLIT>(a, l.logits.shape, l.staged, s);
  }
  // few rows: more lanes each, so that no lane walks many tiles (16 rows of 512 tiles: 14 us with 16 lanes a row); many rows:
  // more of them a block, so that fewer sums are left
  auto rows = [&](auto kernel, int per_block, int threads) {
    const unsigned blocks = (unsigned)ceil_div(d->rows, per_block);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, s, (const float2*)f.partial, l.rows_padded, tiles,
                       (const float*)f.target_logit, d->target, d->ignore_index, d->vocab, d->z_loss, d->rows, row_loss, stats,
                       d->reduction, f.pairs, loss, divisor);
    if (d->reduction != VSL_REDUCE_NONE && blocks > 1) launch_sum_pairs(f.pairs, blocks, d->reduction, loss, divisor, s);
  };
  if (d->rows <= 64 && tiles <= 64) rows(k_ce_rows<64, 1024>, 64, 1024);
  else if (tiles > 64 && d->rows <= 2048) rows(k_ce_rows<4, kThreads>, 4, kThreads);
  else if (d->rows >= 32768 || tiles <= 16) rows(k_ce_rows<64, kThreads>, 64, kThreads);
  else rows(k_ce_rows<16, kThreads>, 16, kThreads);
}

template <typename T, bool SPLIT>
void run_backward(const vsl_linear_ce_desc* d, const Backward& b, const float* stats, const float* divisor, const float* g_loss,
                  T* grad_hidden, T* grad_weight, T* grad_bias, hipStream_t s) {
  typedef std::conditional_t<SPLIT, __bf16, T> O;
  const Layout& l = b.l;
  // float16 keeps 2^-14 as its smallest normal number: with the largest gradient at 2^12 (a derivative is at most that) a
  // probability down to 2^-26 keeps all its bits
  const float unit = __is_same(T, _Float16) ? 4096.0f : 1.0f;
  const float* mean_of = d->reduction == VSL_REDUCE_MEAN ? divisor : nullptr;
  const bool uniform = d->reduction != VSL_REDUCE_NONE && d->z_loss == 0.0f;
  const float* row_scale = uniform ? nullptr : b.row_scale;
  const float* row_size = uniform ? nullptr : b.row_size;
  const OutScale scale = uniform ? OutScale{g_loss, mean_of, nullptr, nullptr, unit}
                                 : OutScale{nullptr, nullptr, b.out_scale, nullptr, unit};
  if (!uniform) {
    ScaleArgs sc{};
    sc.g_loss = g_loss;
    sc.divisor = mean_of;
    sc.stats = stats;
    sc.target = d->target;
    sc.ignore_index = d->ignore_index;
    sc.rows = d->rows;
    sc.rows_padded = l.rows_padded;
    sc.per_row = d->reduction == VSL_REDUCE_NONE;
    sc.z_loss = d->z_loss;
    sc.unit = unit;
    sc.row_scale = b.row_scale;
    sc.row_size = b.row_size;
    sc.out_scale = b.out_scale;
    const int64_t n = ceil_div(d->rows, kThreads);
    sc.partial = b.largest;
    sc.partials = (int)(n > 256 ? 256 : n);
    hipLaunchKernelGGL(k_ce_largest, dim3(sc.partials), dim3(kThreads), 0, s, sc);
    hipLaunchKernelGGL(k_ce_scale, dim3((unsigned)ceil_div(l.rows_padded, kThreads)), dim3(kThreads), 0, s, sc);
  }
  const O* hidden = (const O*)(l.copy_hidden ? b.hidden : d->hidden);
  const int64_t ldh = l.copy_hidden ? l.planes * l.dim_padded : d->hidden_stride;
  const int64_t ldw = l.copy_weight ? l.planes * l.dim_padded : d->weight_stride;
  for (int64_t p = 0; p < b.pieces; ++p) {
    const int64_t v0 = p * b.piece, classes = d->vocab - v0 < b.piece ? d->vocab - v0 : b.piece;
    const T* given = (const T*)d->weight + v0 * d->weight_stride;
    const T* bias = d->bias ? (const T*)d->bias + v0 : nullptr;
    int shape = b.pieces == 1 ? l.logits.shape : plan_of(classes, d->rows, l.steps(d->dim), l.type, false, l.staged).shape;
    if (sizeof(O) == 2 && shape == kThin) shape = kNarrow;
    // what the derivative kernel covers: whole steps of K (32 float32, 64 in 16 bits) for the two products that follow
    const int64_t padded = round_up(classes, b.parts ? 64 : kShapes[shape].bm);
    const int64_t rows_covered = round_up(d->rows, b.parts ? 64 : kShapes[shape].bn);
    LayoutLaunch lay;
    if (p == 0) {
      if (l.copy_hidden) lay.copy(d->hidden, d->hidden_stride, d->rows, d->dim, l.dim_padded, b.hidden);
      if (grad_weight)
        lay.transpose(d->hidden, d->hidden_stride, d->rows, d->dim, l.rows_padded, l.rows_padded,
                      Contributes{d->target, stats, row_scale, nullptr, d->ignore_index}, b.hidden_t);
    }
    if (l.copy_weight) lay.copy(given, d->weight_stride, classes, d->dim, l.dim_padded, b.weight);
    if (grad_hidden && !b.columns)
      lay.transpose(given, d->weight_stride, classes, d->dim, b.piece, padded, Contributes{nullptr, nullptr, nullptr, bias, 0},
                    b.weight_t);
    lay.run<T, SPLIT>(s);
    LogitArgs a{};
    a.op = {l.copy_weight ? b.weight : (const void*)given, hidden, ldw, ldh, (int)classes, (int)d->rows,
            (int)(l.dim_padded / Kind<O>::BK), l.dim_padded, l.dim_padded, l.tail, (int)d->dim};
    if constexpr (SPLIT) a.given_a = given, a.given_b = (const T*)d->hidden;
    a.given_lda = d->weight_stride;
    a.given_ldb = d->hidden_stride;
    a.bias = d->bias;
    a.target = d->target;
    a.class0 = v0;
    a.rows_padded = l.rows_padded;
    a.stats = stats;
    a.row_scale = row_scale;
    a.row_size = row_size;
    a.out_scale = b.out_scale;
    a.unit = unit;
    a.ignore_index = d->ignore_index;
    a.z_loss = d->z_loss;
    a.delta = grad_hidden ? b.delta : nullptr;
    a.ldd = l.planes * b.piece;
    a.plane_d = b.piece;
    a.ldt = l.planes * l.rows_padded;
    a.delta_t = grad_weight || grad_bias ? b.delta_t : nullptr;
    bool made = false;
    if constexpr (!SPLIT)
      if (b.parts) {
        launch_parts<T>(a.op, l, b.parts, s);
        hipLaunchKernelGGL(k_ce_parts_delta<T>, dim3((unsigned)(padded / 64), (unsigned)(rows_covered / kPartRows)), dim3(kThreads),
                           0, s, Parts{b.parts, l.logits.splits, d->rows, d->vocab, d->bias}, a);
        made = true;
      }
    if (!made) {
      if (uniform) launch_logits<T, kDerivatives, SPLIT>(a, shape, l.staged, s);
      else launch_logits<T, kRowDerivatives, SPLIT>(a, shape, l.staged, s);
    }
    GradArgs g[2] = {};
    int shapes[2], n = 0;
    FinishLaunch finish;
    if (grad_hidden) {
      g[n].op = {b.weight_t, b.delta, l.planes * b.piece, l.planes * b.piece, (int)d->dim, (int)d->rows,
                 (int)(padded / Kind<O>::BK), b.piece, b.piece, 8, 0};
      g[n].add = p > 0;
      g[n].sum = b.sum_h;
      g[n].out = grad_hidden;
      g[n].scale = scale;
      g[n].scale.rows = row_size;
      g[n].splits = b.plan_h.splits;
      shapes[n++] = b.plan_h.shape;
      if (b.columns) {
        g[0].op.A = given;
        g[0].op.lda = d->weight_stride;
        g[0].op.rows_of_k = (int)classes;
        g[0].whole = d->dim % 4 == 0;
        g[0].op.bias = bias;
      }
      if (b.sum_h && p == b.pieces - 1)
        finish.add(b.sum_h, b.plan_h.splits, d->rows * d->dim, grad_hidden, row_size, d->dim);
    }
    if (grad_weight) {
      g[n].op = {b.hidden_t, b.delta_t, l.planes * l.rows_padded, l.planes * l.rows_padded, (int)d->dim, (int)classes,
                 (int)(rows_covered / Kind<O>::BK), l.rows_padded, l.rows_padded, 8, 0};
      g[n].sum = b.sum_w;
      g[n].out = grad_weight + v0 * d->dim;
      g[n].scale = scale;
      g[n].splits = b.plan_w.splits;
      shapes[n++] = b.plan_w.shape;
      if (b.sum_w) finish.add(b.sum_w, b.plan_w.splits, classes * d->dim, grad_weight + v0 * d->dim);
    }
    int first = 0;
    if constexpr (!SPLIT)
      if (b.columns) {
        if (shapes[0] == kThin) launch_grad_as<T, Thin, false, kStagedColumns>(g, 1, s);
        else if (shapes[0] == kNarrow) launch_grad_as<T, Narrow, false, kStagedColumns>(g, 1, s);
        else launch_grad_as<T, Small, false, kStagedColumns>(g, 1, s);
        first = 1;
      }
    launch_grad<T, SPLIT>(g + first, shapes + first, n - first, s);
    if (grad_bias) {
      // few classes: their rows in parts, so that more than a block per class works on them
      const int parts = b.sum_b ? (int)(kBiasBlocks / classes < 1 ? 1 : kBiasBlocks / classes) : 1;
      auto sum_rows = [&](auto kernel, int per_block) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(classes * parts, per_block)), dim3(kThreads), 0, s,
                           (const void*)b.delta_t, l.planes * l.rows_padded, l.rows_padded, rows_covered, (int)classes, parts,
                           parts > 1 ? b.sum_b : nullptr, scale, grad_bias + v0);
      };
      // few rows: a block per class would have little to add up (57 rows, 90227 classes: 58 us, with 8 lanes 5)
      if (rows_covered <= 1024) sum_rows(k_ce_bias<T, SPLIT, 8>, kThreads / 8);
      else sum_rows(k_ce_bias<T, SPLIT, kThreads>, 1);
      if (parts > 1) finish.add(b.sum_b, parts, classes, grad_bias + v0);
    }
    finish.run<T>(scale, !uniform, s);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_zero(T* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) p[i] = (T)0.0f;
}
// no rows: the gradients of the shared operands are zero
template <typename T>
void zero_shared(const vsl_linear_ce_desc* d, void* grad_weight, void* grad_bias, hipStream_t s) {
  if (grad_weight)
    hipLaunchKernelGGL(k_zero<T>, linear_grid(d->vocab * d->dim), dim3(kThreads), 0, s, (T*)grad_weight, d->vocab * d->dim);
  if (grad_bias) hipLaunchKernelGGL(k_zero<T>, linear_grid(d->vocab), dim3(kThreads), 0, s, (T*)grad_bias, d->vocab);
}

int check_space(const void* workspace, size_t have, size_t need) {
  if (have < need) return fail(VSL_ERR_WORKSPACE_TOO_SMALL, "linear_ce: workspace too small");
  if (need && (!workspace || (uintptr_t)workspace % 256))
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: workspace must be 256-byte aligned and not NULL");
  return VSL_OK;
}

}  // namespace
}  // namespace vsl_vocab

using namespace vsl_vocab;

extern "C" {

size_t vsl_linear_ce_fwd_workspace_bytes(const vsl_linear_ce_desc* d) {
  return check_ce(d) ? 0 : forward_workspace(d, nullptr).total;
}

int vsl_linear_ce_fwd(const vsl_linear_ce_desc* d, float* row_loss, float* stats, float* loss, float* divisor, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (int rc = check_ce(d)) return rc;
  if (d->rows > 0 && (!row_loss || !stats)) return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: NULL output");
  if (d->reduction != VSL_REDUCE_NONE && (!loss || !divisor)) return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce: NULL loss");
  const Forward f = forward_workspace(d, workspace);
  if (int rc = check_space(workspace, workspace_bytes, f.total)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (d->rows == 0) {
    if (d->reduction != VSL_REDUCE_NONE) launch_sum_pairs(f.pairs, 0, d->reduction, loss, divisor, s);
  } else {
    auto run = d->type == VSL_TYPE_BF16 ? run_forward<__bf16, false> : d->type == VSL_TYPE_F16 ? run_forward<_Float16, false>
               : f.l.split ? run_forward<float, true> : run_forward<float, false>;
    run(d, f, row_loss, stats, loss, divisor, s);
  }
  return launch_status("linear_ce");
}

size_t vsl_linear_ce_bwd_workspace_bytes(const vsl_linear_ce_desc* d, uint32_t grad_mask) {
  return check_ce(d) || d->rows == 0 ? 0 : backward_workspace(d, grad_mask, nullptr).total;
}

int vsl_linear_ce_bwd(const vsl_linear_ce_desc* d, const float* stats, const float* divisor, const float* g_loss, void* grad_hidden,
                      void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_ce(d)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (d->rows == 0) {
    if (d->type == VSL_TYPE_F32) zero_shared<float>(d, grad_weight, grad_bias, s);
    else zero_shared<_Float16>(d, grad_weight, grad_bias, s);  // zero has the same bits in both 16-bit types
    return launch_status("linear_ce backward");
  }
  if (!stats || !g_loss || (d->reduction == VSL_REDUCE_MEAN && !divisor))
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce backward: NULL tensor");
  if (!grad_hidden && !grad_weight && !grad_bias) return VSL_OK;
  const int size = size_of(d->type);
  if ((uintptr_t)grad_hidden % size || (uintptr_t)grad_weight % size || (uintptr_t)grad_bias % size)
    return fail(VSL_ERR_INVALID_ARGUMENT, "linear_ce backward: misaligned gradient");
  const uint32_t mask = (grad_hidden ? 1u : 0u) | (grad_weight ? 2u : 0u) | (grad_bias ? 4u : 0u);
  const Backward b = backward_workspace(d, mask, workspace);
  if (int rc = check_space(workspace, workspace_bytes, b.total)) return rc;
  if (d->type == VSL_TYPE_F32)
    (b.l.split ? run_backward<float, true> : run_backward<float, false>)(d, b, stats, divisor, g_loss, (float*)grad_hidden,
                                                                         (float*)grad_weight, (float*)grad_bias, s);
  else if (d->type == VSL_TYPE_BF16)
    run_backward<__bf16, false>(d, b, stats, divisor, g_loss, (__bf16*)grad_hidden, (__bf16*)grad_weight, (__bf16*)grad_bias, s);
  else
    run_backward<_Float16, false>(d, b, stats, divisor, g_loss, (_Float16*)grad_hidden, (_Float16*)grad_weight, (_Float16*)grad_bias, s);
  return launch_status("linear_ce backward");
}

}  // extern "C"
