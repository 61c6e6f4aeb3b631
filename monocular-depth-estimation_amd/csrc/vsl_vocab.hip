// libvsloss.so -- losses over a set of classes, the part that works on logits in hand: the k largest logits of every row
// (what a teacher hands on) and the distillation of a student from them, forward and backward; and the reduction of row
// losses that the linear cross entropy (vsl_linear_ce.hip) shares.
//
// A row is a token over a large vocabulary or a pixel over its depth bins, so there are two programs for each operator:
// "rows" keeps a whole short row in the registers of 8, 16 or 64 lanes, "stream" walks a long row, or a segment of it when
// there are few rows, with a running maximum and sum per thread.  Both read every logit once per direction.
#include "vsl_vocab.hpp"

namespace vsl_vocab {

static_assert(sizeof(vsl_top_desc) == 48 && sizeof(vsl_distill_desc) == 88, "C-ABI struct layout changed");

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMaxBlocks = 1 << 20;  // blocks of one launch; kernels walk further items in steps of the grid

// ------------------------------------------------------------------------------------------------------------------
// reduced loss
// ------------------------------------------------------------------------------------------------------------------
constexpr int kSumBlocks = 1024;
constexpr int64_t kSumRows = 1024;  // rows a block of the first pass takes at least
constexpr int kFinalThreads = 1024;

template <int WAVES>
__device__ __forceinline__ void block_sum2(double& a, double& b, double* red) {
  for (int m = 32; m >= 1; m >>= 1) {
    a += __shfl_xor(a, m, 64);
    b += __shfl_xor(b, m, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    red[2 * (threadIdx.x >> 6)] = a;
    red[2 * (threadIdx.x >> 6) + 1] = b;
  }
  __syncthreads();
  a = b = 0.0;
  for (int w = 0; w < WAVES; ++w) {
    a += red[2 * w];
    b += red[2 * w + 1];
  }
}

// Sums of losses and weights in double, in an order that depends on the rows alone: 4 and 3 us.
__global__ __launch_bounds__(kThreads) void k_sum_rows(const float* __restrict__ row_loss, const float* __restrict__ weights,
                                                       int64_t rows, int64_t per_block, int reduction,
                                                       double* __restrict__ partial, float* __restrict__ loss,
                                                       float* __restrict__ divisor) {
  __shared__ double red[2 * kWaves];
  const int64_t r0 = blockIdx.x * per_block, r1 = min(rows, r0 + per_block);
  double total = 0.0, count = 0.0;
  for (int64_t r = r0 + threadIdx.x; r < r1; r += kThreads) {
    total += (double)row_loss[r];
    count += weights ? (double)weights[r] : 1.0;
  }
  block_sum2<kWaves>(total, count, red);
  if (threadIdx.x) return;
  if (gridDim.x == 1) {
    finish_sum(total, count, reduction, loss, divisor);
  } else {
    partial[2 * blockIdx.x] = total;
    partial[2 * blockIdx.x + 1] = count;
  }
}

__global__ __launch_bounds__(kFinalThreads) void k_sum_final(const double* __restrict__ pairs, int64_t n, int reduction,
                                                             float* __restrict__ loss, float* __restrict__ divisor) {
  __shared__ double red[2 * (kFinalThreads / 64)];
  double total = 0.0, count = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kFinalThreads) {
    total += pairs[2 * i];
    count += pairs[2 * i + 1];
  }
  block_sum2<kFinalThreads / 64>(total, count, red);
  if (threadIdx.x == 0) finish_sum(total, count, reduction, loss, divisor);
}

int sum_blocks(int64_t rows) {
  const int64_t b = ceil_div(rows, kSumRows);
  return (int)(b < 1 ? 1 : (b > kSumBlocks ? kSumBlocks : b));
}

}  // namespace

size_t sum_workspace_bytes(int64_t rows) { return up256((size_t)sum_blocks(rows) * 2 * sizeof(double)); }

void launch_sum(const float* row_loss, const float* weights, int64_t rows, int reduction, void* partial, float* loss,
                float* divisor, hipStream_t s) {
  const int n = sum_blocks(rows);
  hipLaunchKernelGGL(k_sum_rows, dim3(n), dim3(kThreads), 0, s, row_loss, weights, rows, ceil_div(rows, n), reduction,
                     (double*)partial, loss, divisor);
  if (n > 1) launch_sum_pairs((const double*)partial, n, reduction, loss, divisor, s);
}
void launch_sum_pairs(const double* pairs, int64_t n, int reduction, float* loss, float* divisor, hipStream_t s) {
  hipLaunchKernelGGL(k_sum_final, dim3(1), dim3(kFinalThreads), 0, s, pairs, n, reduction, loss, divisor);
}

namespace {

// ------------------------------------------------------------------------------------------------------------------
// keys: unsigned integers that order as (value, lower index first); 0 is below every key of an element
// ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned ordered32(unsigned b) {
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;  // NaN: above +infinity
  if (b == 0x80000000u) b = 0u;                             // -0 ties with +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr unsigned kOrderedLowest = 0x007FFFFFu;            // -infinity
__device__ __forceinline__ unsigned unordered32(unsigned o) { return o & 0x80000000u ? o & 0x7FFFFFFFu : ~o; }

// Short rows: a 16-bit value as a float has at least 13 zero bits at the end, so value and index share 32 bits; float32
// takes 64.  make: a NaN has to be a positive one (which orders above +infinity), the callers see to it.
template <typename T>
struct RowKey {
  typedef unsigned K;
  static constexpr unsigned kIndex = 2047u;  // a short row has at most 2048 classes
  static __device__ __forceinline__ K make(float x, int index) {
    const unsigned b = __float_as_uint(x + 0.0f);  // -0 ties with +0
    const unsigned o = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
    return (o & ~kIndex) | (kIndex - (unsigned)index);
  }
  static __device__ __forceinline__ int index(K k) { return (int)(kIndex - (k & kIndex)); }
  static __device__ __forceinline__ T value(K k) {
    const unsigned o = k & ~kIndex;
    return (T)__uint_as_float((o & 0x80000000u ? o & 0x7FFFFFFFu : ~o) & ~kIndex);
  }
};
template <>
struct RowKey<float> {
  typedef unsigned long long K;
  static __device__ __forceinline__ K make(float x, int index) {
    return (unsigned long long)ordered32(__float_as_uint(x)) << 32 | (0xFFFFFFFFu - (unsigned)index);
  }
  static __device__ __forceinline__ int index(K k) { return (int)(0xFFFFFFFFu - (unsigned)k); }
  static __device__ __forceinline__ float value(K k) { return __uint_as_float(unordered32((unsigned)(k >> 32))); }
};

// ------------------------------------------------------------------------------------------------------------------
// top logits
// ------------------------------------------------------------------------------------------------------------------
struct TopArgs {
  const void* logits;
  void* values;
  int* indices;
  float* lse;
  unsigned long long* keys;  // [rows][segs][k], stream only
  float* stat;               // [rows][segs][2] running maximum and sum, stream only
  int64_t rows, stride;
  int V, k, segs, seg_len;
  float c, inv_t;            // log2(e) / temperature, 1 / temperature
};

// A lane's own keys, larger first: the odd-even merge network, N a power of two.
template <int N, typename K>
__device__ __forceinline__ void sort_own(K (&key)[N]) {
#pragma unroll
  for (int p = 1; p < N; p <<= 1)
#pragma unroll
    for (int q = p; q >= 1; q >>= 1)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const K a = key[i + j], b = key[i + j + q];
            key[i + j] = a > b ? a : b;
            key[i + j + q] = a > b ? b : a;
          }
}

// The sorted keys of the L lanes of a group, as one list, N to a lane: bitonic merges of twice as many lanes each, first
// against the other half in reverse, then over half the distance and so on down to the lane's own keys.
template <int S, typename K, int N>
__device__ __forceinline__ void exchange(K (&key)[N]) {  // with lane ^ S (a power of two): the lower lane keeps the larger ones
  const bool upper = threadIdx.x & S;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const K other = lane_xor<S>(key[e]);
    key[e] = (other > key[e]) != upper ? other : key[e];
  }
}
template <int S, typename K, int N>
__device__ __forceinline__ void merge_lanes(K (&key)[N]) {  // two lists of S / 2 lanes each
  const bool upper = threadIdx.x & (S / 2);
  K other[N];
#pragma unroll
  for (int e = 0; e < N; ++e) other[e] = lane_xor<S - 1>(key[N - 1 - e]);
#pragma unroll
  for (int e = 0; e < N; ++e) key[e] = (other[e] > key[e]) != upper ? other[e] : key[e];
  if (S >= 64) exchange<16>(key);
  if (S >= 32) exchange<8>(key);
  if (S >= 16) exchange<4>(key);
  if (S >= 8) exchange<2>(key);
  if (S >= 4) exchange<1>(key);
#pragma unroll
  for (int q = N / 2; q >= 1; q >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!(i & q)) {
        const K a = key[i], b = key[i + q];
        key[i] = a > b ? a : b;
        key[i + q] = a > b ? b : a;
      }
}
template <int L, typename K, int N>
__device__ __forceinline__ void merge_group(K (&key)[N]) {
  merge_lanes<2>(key);
  merge_lanes<4>(key);
  merge_lanes<8>(key);
  if (L > 8) merge_lanes<16>(key);
  if (L > 16) {
    merge_lanes<32>(key);
    merge_lanes<64>(key);
  }
}

// The eight largest of a lane's keys, larger first, and of a group's, which every lane gets: of two sorted lists the larger
// of each place and its mirror are the largest eight, in bitonic order.
template <typename K>
__device__ __forceinline__ void clean8(K (&key)[8]) {
#pragma unroll
  for (int q = 4; q >= 1; q >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(i & q)) {
        const K a = key[i], b = key[i + q];
        key[i] = a > b ? a : b;
        key[i + q] = a > b ? b : a;
      }
}
template <int N, typename K>
__device__ __forceinline__ void own_top8(const K (&key)[N], K (&best)[8]) {
#pragma unroll
  for (int c = 0; c < (N + 7) / 8; ++c) {
    K part[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) part[e] = 8 * c + e < N ? key[8 * c + e] : (K)0;
    sort_own<8>(part);
#pragma unroll
    for (int e = 0; e < 8; ++e) best[e] = c == 0 || part[7 - e] > best[e] ? part[c == 0 ? e : 7 - e] : best[e];
    if (c > 0) clean8(best);
  }
}
template <int X, typename K>
__device__ __forceinline__ void join_top8(K (&best)[8]) {
  K other[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) other[e] = lane_xor<X>(best[7 - e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) best[e] = other[e] > best[e] ? other[e] : best[e];
  clean8(best);
}
template <int L, typename K>
__device__ __forceinline__ void group_top8(K (&best)[8]) {  // mirrors: after every step all lanes of a half hold the same
  join_top8<1>(best);
  join_top8<3>(best);
  join_top8<7>(best);
  if (L > 8) join_top8<15>(best);
  if (L > 16) {
    join_top8<31>(best);
    join_top8<63>(best);
  }
}

// Short rows: L lanes hold NV vectors each.  Up to eight keys (kEight): lists of eight are joined over the lanes.  Else every
// lane sorts its keys; every round takes the largest of the group's first ones, and its lane moves on to its next (kRounds),
// or, for many keys, the lanes' lists are merged (kMerge).
// 368640 x 96 float16, k = 8: 34 us, 2.6 TB/s; bound by the vector instructions of the sorts.
enum { kEight, kRounds, kMerge };
template <typename T, int L, int NV, int FORM>
__global__ __launch_bounds__(kThreads) void k_top_rows(TopArgs a) {
  constexpr int E = Vec<T>::E, G = kThreads / L;
  typedef typename RowKey<T>::K K;
  const int lane = threadIdx.x % L;
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += (int64_t)gridDim.x * G) {
    const int64_t row = r0 + threadIdx.x / L;
    const bool live = row < a.rows;  // whole groups: the lanes of a group agree
    const T* x = (const T*)a.logits + (live ? row : 0) * a.stride;
    float xs[NV][E];
    MaxSum t{ninf(), 0.0f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (v * L + lane) * E;
      unpack(load_row(x, i, i < a.V ? a.V : i), xs[v], (const T*)nullptr);
#pragma unroll
      for (int e = 0; e < E; ++e) t.m = __builtin_elementwise_maximum(t.m, xs[v][e]);
    }
    if (__any(t.m != t.m)) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) xs[v][e] = xs[v][e] != xs[v][e] ? qnan() : xs[v][e];
    }
    K key[NV * E];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = (v * L + lane) * E + e;
        key[v * E + e] = i < a.V ? RowKey<T>::make(xs[v][e], i) : (K)0;
      }
    if (a.lse) {
      t.m = group_all<L>(t.m, MaxF());
      const Exponent ex(exp_ref(t.m), a.c);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) t.s += ex(xs[v][e]);
      t.s = group_all<L>(t.s, AddF()) * ex.factor();
      if (live && lane == 0) a.lse[row] = log_sum(t, a.inv_t);
    }
    if (FORM == kEight) {
      K best[8];
      own_top8<NV * E>(key, best);
      group_top8<L>(best);
      if (live && lane < a.k) {
        K mine = best[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mine = lane == e ? best[e] : mine;
        ((T*)a.values)[row * a.k + lane] = RowKey<T>::value(mine);
        a.indices[row * a.k + lane] = RowKey<T>::index(mine);
      }
      continue;
    }
    sort_own<NV * E>(key);
    if (FORM == kMerge) {
      merge_group<L>(key);
#pragma unroll
      for (int e = 0; e < NV * E; ++e) {
        const int j = lane * NV * E + e;
        if (live && j < a.k) {
          ((T*)a.values)[row * a.k + j] = RowKey<T>::value(key[e]);
          a.indices[row * a.k + j] = RowKey<T>::index(key[e]);
        }
      }
      continue;
    }
    K mine = 0;
    for (int j = 0; j < a.k; ++j) {
      const K best = group_all<L>(key[0], MaxU());
      const bool taken = key[0] == best;  // by one lane: no key occurs twice, and 0 follows the last
#pragma unroll
      for (int e = 0; e < NV * E - 1; ++e) key[e] = taken ? key[e + 1] : key[e];
      key[NV * E - 1] = taken ? (K)0 : key[NV * E - 1];
      if (j % L == lane) mine = best;
      if ((j % L == L - 1 || j == a.k - 1) && live && lane <= j % L) {
        const int64_t at = row * a.k + j - j % L + lane;
        ((T*)a.values)[at] = RowKey<T>::value(mine);
        a.indices[at] = RowKey<T>::index(mine);
      }
    }
  }
}

// Long rows, kGroup vectors a thread at a time, the next ones under way meanwhile.  A key is (ordered value, ~index).
// First only the threads' maxima over the first kProbe groups are taken: their k-th largest is a bound that at least k
// elements reach.  Then, from the start (what was read is in L2 still), the elements that reach the bound are collected,
// and whenever more than `trigger` are there the k largest of them are kept and the bound rises to the k-th.  A group of
// which more passes than the buffer holds (rising rows) is collected again, vector by vector.
// 4096 x 131072 bfloat16, k = 64: 268 us, 4.0 TB/s read, vector instructions 75 % busy; 1 x 50021, k = 32: 10 us, latency.
constexpr int kProbe = 4;
constexpr int kGroup = 2;
constexpr int kTrigger = 512;  // at most; see trigger below
constexpr int kBuffer = 4096;  // kTrigger + one vector of each thread, as a power of two for the sort
static_assert(kTrigger + kThreads * 8 <= kBuffer && VSL_MAX_TOP <= kTrigger, "candidate buffer");

// Bitonic sort, larger first, of 256 R keys: thread t holds keys t, t + 256, ...  Partners within a wave trade by
// shuffles, within a thread by registers; only strides of 64 and 128 go through LDS and barriers.
template <int R>
__device__ __forceinline__ void sort_step(unsigned long long (&key)[R], unsigned long long* lds, int size, int step) {
  const int tid = threadIdx.x;
  if (R > 1 && step >= kThreads) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int o = r + step / kThreads;
      if ((r * kThreads) & step || o >= R) continue;
      const unsigned long long u = key[r], v = key[o];
      const bool keep = (u > v) == (((r * kThreads) & size) == 0);
      key[r] = keep ? u : v;
      key[o] = keep ? v : u;
    }
    return;
  }
  unsigned long long other[R];
  if (step >= 64) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) lds[r * kThreads + tid] = key[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) other[r] = lds[r * kThreads + (tid ^ step)];
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) other[r] = __shfl_xor(key[r], step, 64);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = r * kThreads + tid;
    const bool take_larger = ((i & size) == 0) == ((i & step) == 0);
    key[r] = (other[r] > key[r]) == take_larger ? other[r] : key[r];
  }
}
template <int R>
__device__ __forceinline__ void sort_registers(unsigned long long (&key)[R], unsigned long long* lds) {
#pragma unroll
  for (int size = 2; size <= kThreads * R; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step >= 1; step >>= 1) sort_step<R>(key, lds, size, step);
}
template <int R>
__device__ __forceinline__ void sort_some(unsigned long long* buf, int count) {
  unsigned long long key[R];
#pragma unroll
  for (int r = 0; r < R; ++r) key[r] = r * kThreads + (int)threadIdx.x < count ? buf[r * kThreads + threadIdx.x] : 0ull;
  sort_registers<R>(key, buf);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) buf[r * kThreads + threadIdx.x] = key[r];
  __syncthreads();
}
// Up to 256 different keys: a key's place is the number of larger ones, which every thread counts for its own key over
// LDS reads that all lanes share.  No step waits for the one before: 2 us less than the bitonic network for 50 keys, 1 us
// for 200.
__device__ __forceinline__ void sort_by_rank(unsigned long long* buf, int count) {
  const int tid = threadIdx.x;
  const unsigned long long key = tid < count ? buf[tid] : 0ull;
  if (tid == 0 && (count & 1)) buf[count] = 0ull;
  __syncthreads();
  int place = 0;
  if ((tid & ~63) < count) {
    const u64x2* pairs = (const u64x2*)buf;
#pragma unroll 4
    for (int j = 0; j < (count + 1) / 2; ++j) {
      const u64x2 two = pairs[j];
      place += (int)(two.x > key) + (int)(two.y > key);
    }
  }
  __syncthreads();
  buf[tid < count ? place : tid] = key;
  __syncthreads();
}
// Sorts the first `count` keys of an LDS buffer of kBuffer, larger first, zeros behind (as far as a power of two or 256).
// Starts behind a barrier that made the keys visible; ends with one.
__device__ __forceinline__ void sort_count(unsigned long long* buf, int count) {
  if (count <= kThreads) return sort_by_rank(buf, count);
  if (count <= 2 * kThreads) return sort_some<2>(buf, count);
  int n = 4 * kThreads;
  while (n < count) n <<= 1;
  for (int i = count + threadIdx.x; i < n; i += kThreads) buf[i] = 0ull;
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step >= 1; step >>= 1) {
      __syncthreads();
      for (int p = threadIdx.x; p < n / 2; p += kThreads) {
        const int i = 2 * p - (p & (step - 1)), j = i + step;
        const unsigned long long u = buf[i], v = buf[j];
        if ((u < v) == ((i & size) == 0)) {
          buf[i] = v;
          buf[j] = u;
        }
      }
    }
  __syncthreads();
}

__device__ __forceinline__ float key_floor(unsigned long long key) {
  // a float that no element of a key >= `key` lies below; NaN keys: +infinity (a NaN is not below it)
  const unsigned o = (unsigned)(key >> 32);
  return o == 0u ? ninf() : o > 0xFF800000u ? __uint_as_float(0x7F800000u) : __uint_as_float(unordered32(o));
}

// N vectors of a thread, kThreads vectors apart
template <typename T, int N>
__device__ __forceinline__ void load_group(const T* x, int i0, int end, u32x4 (&r)[N]) {
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int i = i0 + (u * kThreads + (int)threadIdx.x) * Vec<T>::E;
    r[u] = load_row(x, i, i < end ? end : i);
  }
}
// running maximum and sum over a group; returns the group's maximum
template <typename T, int N>
__device__ __forceinline__ float add_group(const float (&v)[N][Vec<T>::E], RunSum& t, float c) {
  float top = v[0][0];
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int e = 0; e < Vec<T>::E; ++e) top = __builtin_elementwise_maximum(top, v[u][e]);
  const Exponent ex = t.move(__builtin_elementwise_maximum(t.m, top), c);
  float s2 = 0.0f;
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int e = 0; e < Vec<T>::E; e += 2) {
      t.s += ex(v[u][e]);
      s2 += ex(v[u][e + 1]);
    }
  t.s += s2;
  return top;
}

template <typename T>
__global__ __launch_bounds__(kThreads, 4) void k_top_stream(TopArgs a) {
  constexpr int E = Vec<T>::E, kSpan = kThreads * E * kGroup;
  __shared__ alignas(16) unsigned long long buf[kBuffer];
  __shared__ int count;
  __shared__ unsigned found;
  __shared__ float red[2 * kWaves];
  const int tid = threadIdx.x;
  const int64_t items = a.rows * a.segs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = item / a.segs;
    const int seg = (int)(item % a.segs);
    const T* x = (const T*)a.logits + row * a.stride;
    const int e0 = seg * a.seg_len, e1 = min(a.V, e0 + a.seg_len);  // a segment never starts behind the row
    RunSum run;
    unsigned long long bound = 0;
    float floor_value = ninf();
    int kept = 0;  // keys in the buffer, as every thread knows it
    const int trigger = min(kTrigger, a.k + max(a.k, 64));  // sorting a few keys is cheaper than collecting by a loose bound
    auto collect = [&](const float (&v)[E], int i) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(v[e] < floor_value)) {  // few lanes, and soon hardly any
          const unsigned long long key = RowKey<float>::make(v[e], i + e);
          if (key >= bound && i + e < e1) {
            const int at = atomicAdd(&count, 1);
            if (at < kBuffer) buf[at] = key;
          }
        }
    };
    auto settle = [&]() {  // everyone has collected: take the count, keep the k largest if there are many
      __syncthreads();
      kept = count;
      __syncthreads();
      if (kept <= trigger || kept > kBuffer) return;
      sort_count(buf, kept);
      bound = buf[a.k - 1] + 1;  // its element is kept: later ones have to be above it
      floor_value = key_floor(bound);
      if (tid == 0) count = a.k;
      kept = a.k;
      __syncthreads();
    };
    u32x4 next[kGroup];
    const int probe_end = min(e1, e0 + kProbe * kSpan);
    load_group(x, e0, e1, next);
    float best = ninf();
    for (int i0 = e0; i0 < probe_end; i0 += kSpan) {
      float v[kGroup][E];
#pragma unroll
      for (int u = 0; u < kGroup; ++u) unpack(next[u], v[u], (const T*)nullptr);
      if (i0 + kSpan < probe_end) load_group(x, i0 + kSpan, e1, next);
      best = __builtin_elementwise_maximum(best, add_group<T>(v, run, a.c));
    }
    if (e1 - e0 > kSpan) load_group(x, e0, e1, next);  // else it is there still
    {
      // The k-th largest of the maxima, by ranks again, over maxima of `share` threads each as long as twice k of them are
      // left: fewer to count through, for a bound that still no more than 1.4 k elements of random rows reach.  The value's
      // upper 24 bits (an element that equals the maximum reaches that as well) over the thread, so that no two are the
      // same.  A thread without an element says -infinity.
      const int share = a.k <= kThreads / 8 ? 4 : a.k <= kThreads / 4 ? 2 : 1;
      if (share >= 2) best = MaxF()(best, dpp<kXor1>(best));
      if (share == 4) best = MaxF()(best, dpp<kXor2>(best));
      unsigned* maxima = (unsigned*)buf;
      const unsigned mine = (ordered32(__float_as_uint(best)) & ~255u) | (unsigned)((kThreads - 1 - tid) / share);
      if (tid % share == 0) maxima[tid / share] = mine;
      __syncthreads();
      int place = 0;
      const u32x4* four = (const u32x4*)maxima;
#pragma unroll 8
      for (int j = 0; j < kThreads / 4 / share; ++j) {
        const u32x4 m = four[j];
        place += (int)(m.x > mine) + (int)(m.y > mine) + (int)(m.z > mine) + (int)(m.w > mine);
      }
      if (place == a.k - 1) found = mine & ~255u;
      if (tid == 0) count = 0;
      __syncthreads();
      const unsigned low = found;
      bound = (unsigned long long)(low < kOrderedLowest ? kOrderedLowest : low) << 32;
      floor_value = key_floor(bound);
    }
    for (int i0 = e0; i0 < e1; i0 += kSpan) {
      float v[kGroup][E];
#pragma unroll
      for (int u = 0; u < kGroup; ++u) unpack(next[u], v[u], (const T*)nullptr);
      if (i0 + kSpan < e1) load_group(x, i0 + kSpan, e1, next);
      float top = v[0][0];
      if (i0 < probe_end) {
#pragma unroll
        for (int u = 0; u < kGroup; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) top = __builtin_elementwise_maximum(top, v[u][e]);
      } else {
        top = add_group<T>(v, run, a.c);
      }
      const int before = kept;
      if (__any(!(top < floor_value)))
#pragma unroll
        for (int u = 0; u < kGroup; ++u) collect(v[u], i0 + (u * kThreads + tid) * E);
      settle();
      if (kept > kBuffer) {
        if (tid == 0) count = before;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
          collect(v[u], i0 + (u * kThreads + tid) * E);
          settle();
        }
      }
    }
    const int n = kept;
    sort_count(buf, n);
    MaxSum t{ninf(), 0.0f};
    if (a.lse || a.segs > 1) t = block_join<kWaves>(run.get(), red, a.c);
    if (a.segs > 1) {
      if (tid < a.k) a.keys[item * a.k + tid] = tid < n ? buf[tid] : 0ull;
      if (tid == 0) {
        a.stat[2 * item] = t.m;
        a.stat[2 * item + 1] = t.s;
      }
    } else {
      if (tid < a.k) {
        ((T*)a.values)[row * a.k + tid] = (T)RowKey<float>::value(buf[tid]);
        a.indices[row * a.k + tid] = RowKey<float>::index(buf[tid]);
      }
      if (a.lse && tid == 0) a.lse[row] = log_sum(t, a.inv_t);
    }
    __syncthreads();
  }
}

// Joins the segments of a row, at most kJoinKeys keys in lists of k, larger first.  All segments but the last are longer
// than k: the smallest of their q-th keys, q = ceil(k / lists), is reached by at least k keys, and so is the largest of all
// lists' k-th.  What is below is left out; of random rows about 2 k keys stay.  5 lists of 32: 4 us, latency.
constexpr int kJoinKeys = kBuffer;
template <typename T>
__global__ __launch_bounds__(kThreads) void k_top_join(TopArgs a) {
  __shared__ alignas(16) unsigned long long buf[kJoinKeys];
  __shared__ unsigned long long low[2];
  __shared__ int count;
  __shared__ float red[2 * kWaves];
  const int tid = threadIdx.x, lists = a.segs - 1, q = (a.k + lists - 1) / lists;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const unsigned long long* keys = a.keys + row * a.segs * a.k;
    const int n = a.segs * a.k;
    if (tid == 0) {
      low[0] = 0ull;
      low[1] = ~0ull;
      count = 0;
    }
    unsigned long long key[4];  // four at a time, the first ones under way while the bound is made
    auto load_keys = [&](int i0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) key[r] = keys[min(i0 + r * kThreads + tid, n - 1)];
    };
    load_keys(0);
    MaxSum t{ninf(), 0.0f};
    __syncthreads();
    for (int s = tid; s < a.segs; s += kThreads) {
      atomicMax(&low[0], keys[s * a.k + a.k - 1]);
      if (s < lists) atomicMin(&low[1], keys[s * a.k + q - 1]);
      if (a.lse) t = join(t, {a.stat[2 * (row * a.segs + s)], a.stat[2 * (row * a.segs + s) + 1]}, a.c);
    }
    __syncthreads();
    const unsigned long long bound = low[0] > low[1] ? low[0] : low[1];
    for (int i0 = 0; i0 < n; i0 += 4 * kThreads) {
      if (i0 > 0) load_keys(i0);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (i0 + r * kThreads + tid < n && key[r] >= bound && key[r] != 0ull) buf[atomicAdd(&count, 1)] = key[r];
    }
    __syncthreads();
    sort_count(buf, count);
    if (tid < a.k) {
      ((T*)a.values)[row * a.k + tid] = (T)RowKey<float>::value(buf[tid]);
      a.indices[row * a.k + tid] = RowKey<float>::index(buf[tid]);
    }
    if (a.lse) {
      t = block_join<kWaves>(t, red, a.c);
      if (tid == 0) a.lse[row] = log_sum(t, a.inv_t);
    }
    __syncthreads();
  }
}

int vec_of(int type) { return type == VSL_TYPE_F32 ? 4 : 8; }
// a row of at most this many elements stays in registers
int64_t short_row(int type) { return 256 * vec_of(type); }

struct Split {
  int segs, seg_len;
};
// Segments of a long row: enough blocks for the 256 CUs when there are few rows, whole tiles each, `least` at least, and at
// most `most` of them.
Split split_row(int64_t rows, int64_t V, int tile, int least, int most) {
  const int64_t tiles = ceil_div(V, tile);
  int64_t segs = ceil_div(1024, rows < 1 ? 1 : rows);
  if (segs > tiles / least) segs = tiles / least;
  if (segs > most) segs = most;
  if (segs < 1) segs = 1;
  const int64_t per = ceil_div(tiles, segs);
  return {(int)ceil_div(tiles, per), (int)(per * tile)};
}

int grid_of(int64_t items) { return (int)(items < 1 ? 1 : (items > kMaxBlocks ? kMaxBlocks : items)); }

Split top_split(const vsl_top_desc* d) {
  if (d->vocab <= short_row(d->type)) return {1, (int)d->vocab};
  // Up to 16 tiles stay whole, a join costs more (200 x 20000 bf16: 10.0 us, in two segments 13.7), and a segment is no
  // shorter than 4 (1 x 50021 bf16, k = 32: 14.7 us, with 2 27.9, with 8 16.4).
  const int tile = kThreads * vec_of(d->type);
  if (d->vocab <= 16 * tile) return {1, (int)ceil_div(d->vocab, tile) * tile};
  return split_row(d->rows, d->vocab, tile, 4, kJoinKeys / d->k);
}

bool bad_type(int t) { return t != VSL_TYPE_F32 && t != VSL_TYPE_BF16 && t != VSL_TYPE_F16; }

int size_of(int type) { return type == VSL_TYPE_F32 ? 4 : 2; }

int check_matrix(const char* what, const void* logits, int64_t rows, int64_t vocab, int64_t stride, int type) {
  if (bad_type(type)) return fail(VSL_ERR_INVALID_ARGUMENT, std::string(what) + ": unknown element type");
  if (rows < 0 || rows >= (1LL << 31) || vocab < 1 || vocab >= (1LL << 30))
    return fail(VSL_ERR_INVALID_ARGUMENT, std::string(what) + ": need 0 <= rows < 2^31 and 1 <= vocab < 2^30");
  if (stride < vocab || stride >= (1LL << 40))
    return fail(VSL_ERR_INVALID_ARGUMENT, std::string(what) + ": the row stride must be at least vocab");
  if ((uintptr_t)logits % size_of(type)) return fail(VSL_ERR_INVALID_ARGUMENT, std::string(what) + ": misaligned logits");
  return VSL_OK;
}
int check_top(const vsl_top_desc* d) {
  if (!d) return fail(VSL_ERR_INVALID_ARGUMENT, "top_logits: descriptor is null");
  if (int rc = check_matrix("top_logits", d->logits, d->rows, d->vocab, d->stride, d->type)) return rc;
  if (d->k < 1 || d->k > VSL_MAX_TOP || d->k > d->vocab)
    return fail(VSL_ERR_INVALID_ARGUMENT, "top_logits: need 1 <= k <= min(vocab, 256)");
  if (!(d->temperature >= 1e-4f && d->temperature <= 1e4f))
    return fail(VSL_ERR_INVALID_ARGUMENT, "top_logits: temperature must lie in 1e-4..1e4");
  return VSL_OK;
}

// Merging the lanes' lists takes the time of about 20 rounds, of 15 with the 64-bit keys of float32 (by rounds and merged:
// 100000 x 60 bf16, k = 16: 13.0 and 12.0 us; 20000 x 500 bf16, k = 16: 24.3 and 26.5, k = 32: 40.2 and 27.7;
// 20000 x 250 f32, k = 8: 24.1 and 24.9, k = 24: 50.3 and 25.7).
template <typename T>
constexpr int most_rounds() { return sizeof(T) == 4 ? 15 : 20; }
template <typename T, int FORM>
void launch_rows(const TopArgs& a, int nv, hipStream_t s) {
  const dim3 b(kThreads);
  const dim3 g8(grid_of(ceil_div(a.rows, kThreads / 8)));
  const dim3 g16(grid_of(ceil_div(a.rows, kThreads / 16))), g64(grid_of(ceil_div(a.rows, kThreads / 64)));
  if (nv <= 8) hipLaunchKernelGGL((k_top_rows<T, 8, 1, FORM>), g8, b, 0, s, a);
  else if (nv <= 16) hipLaunchKernelGGL((k_top_rows<T, 8, 2, FORM>), g8, b, 0, s, a);
  else if (nv <= 32) hipLaunchKernelGGL((k_top_rows<T, 16, 2, FORM>), g16, b, 0, s, a);
  else if (nv <= 64) hipLaunchKernelGGL((k_top_rows<T, 16, 4, FORM>), g16, b, 0, s, a);
  else if (nv <= 128) hipLaunchKernelGGL((k_top_rows<T, 64, 2, FORM>), g64, b, 0, s, a);
  else hipLaunchKernelGGL((k_top_rows<T, 64, 4, FORM>), g64, b, 0, s, a);
}
template <typename T>
void launch_top(const TopArgs& a, bool rows_program, hipStream_t s) {
  if (rows_program) {
    const int nv = (int)ceil_div(a.V, Vec<T>::E);
    // The join of eights takes the time of about five rounds (by rounds and joined: 368640 x 96 float16, k = 8: 41.2 and 33.9
    // us; 100000 x 60 bfloat16, k = 4: 7.7 and 8.5; 20000 x 250 float32, k = 8: 24.1 and 12.8), of more where 64 lanes trade
    // 64-bit keys and hold few (11261 x 288 float32, k = 7: 16.3 and 20.3).
    const bool eight = a.k >= 5 && a.k <= 8 && !(sizeof(T) == 4 && nv > 64 && nv <= 128);
    if (eight) launch_rows<T, kEight>(a, nv, s);
    else if (a.k > most_rounds<T>()) launch_rows<T, kMerge>(a, nv, s);
    else launch_rows<T, kRounds>(a, nv, s);
    return;
  }
  hipLaunchKernelGGL(k_top_stream<T>, dim3(grid_of(a.rows * a.segs)), dim3(kThreads), 0, s, a);
  if (a.segs > 1) hipLaunchKernelGGL(k_top_join<T>, dim3(grid_of(a.rows)), dim3(kThreads), 0, s, a);
}

// ------------------------------------------------------------------------------------------------------------------
// distillation from top logits
// ------------------------------------------------------------------------------------------------------------------
struct DistillArgs {
  const void* logits;
  const void* values;
  const void* indices;
  const float* lse;
  const float* weights;
  float* row_loss;
  float* stats;        // [rows] of RowStats
  float* partial;      // [rows][segs][2], stream only
  double* sums;        // [blocks][2] weighted losses and weights of a block's rows, short rows only; NULL: not wanted
  const float* divisor;  // backward: of the mean
  const float* g_loss;
  void* grad;
  int64_t rows, stride, grad_stride;
  int V, k, segs, seg_len, value_type, index_bytes, reduction;
  float c;             // log2(e) / temperature
  float ih, il;        // 1 / temperature as a sum of two floats
  float temperature;
};

__device__ __forceinline__ float teacher_value(const DistillArgs& a, int64_t at) {
  if (a.value_type == VSL_TYPE_F32) return ((const float*)a.values)[at];
  if (a.value_type == VSL_TYPE_BF16) return (float)((const __bf16*)a.values)[at];
  return (float)((const _Float16*)a.values)[at];
}
// -1 for an index outside the vocabulary
__device__ __forceinline__ int teacher_index(const DistillArgs& a, int64_t at) {
  const int64_t i = a.index_bytes == 8 ? ((const int64_t*)a.indices)[at] : (int64_t)((const int*)a.indices)[at];
  return i < 0 || i >= a.V ? -1 : (int)i;
}

// log q, kept in two floats: rounded to one it would be off by half an ulp of its size, and that error of every q would land
// in q_t = 1 - sum q, which is small.
struct LogQ {
  float hi, lo;
  __device__ __forceinline__ float log() const { return hi + lo; }
  __device__ __forceinline__ float q() const {
    // hi log2(e) in two floats as well: 2^p (1 + the rest)
    const float p = __fmul_rn(hi, kLog2e), pe = fmaf(hi, kLog2e, -p);
    const float rest = fmaf(fmaf(hi, kLog2eLow, pe), kLn2, lo), e = __builtin_amdgcn_exp2f(p);
    return hi == ninf() ? 0.0f : fmaf(e, rest, e);
  }
};
struct TeacherSum {
  float base, log_sum;  // lse and kWhole where it is given; the largest value itself and the log of the sum above it otherwise
};
constexpr float kWhole = -1.0f;  // a log of a sum whose largest term is 1 is not negative
// v / T - lse, or (v - largest) / T - log_sum: the difference comes first where there is one, since the largest value / T,
// rounded, would be off by half an ulp of its own size in every q
__device__ __forceinline__ LogQ log_q(const DistillArgs& a, float v, TeacherSum t) {
  if (v == ninf()) return {ninf(), 0.0f};
  const bool whole = t.log_sum < 0.0f;
  const float x = whole ? v : v - t.base, base = whole ? t.base : t.log_sum;
  const float p = __fmul_rn(x, a.ih);
  const float pe = fmaf(x, a.il, fmaf(x, a.ih, -p));
  const float s = __fsub_rn(p, base), b = __fsub_rn(s, p);
  return {s, pe + __fadd_rn(__fsub_rn(p, __fsub_rn(s, b)), __fsub_rn(-base, b))};
}

// weight of a row, its share of the upstream gradient and the factor T of the derivative
__device__ __forceinline__ float row_scale(const DistillArgs& a, int64_t row, float w) {
  float g = a.g_loss[a.reduction == VSL_REDUCE_NONE ? row : 0];
  if (a.reduction == VSL_REDUCE_MEAN) {
    const float n = *a.divisor;
    g = n == 0.0f ? 0.0f : g / n;
  }
  return g * w * a.temperature;
}

struct RowStats {
  float m, ls;        // p = 2^((x - m) c - ls); m = +inf: the row adds nothing
  float tm, tls;      // the same over the classes that are not the teacher's
  float qt, total;    // the teacher's rest; sum of all q
  TeacherSum teacher;
  __device__ __forceinline__ void store(const DistillArgs& a, int64_t row) const {
    f32x4* p = (f32x4*)(a.stats + row * VSL_DISTILL_STATS);
    p[0] = f32x4{m, ls, tm, tls};
    p[1] = f32x4{qt, total, teacher.base, teacher.log_sum};
  }
  __device__ __forceinline__ void load(const DistillArgs& a, int64_t row) {
    const f32x4* p = (const f32x4*)(a.stats + row * VSL_DISTILL_STATS);
    const f32x4 u = p[0], v = p[1];
    m = u[0], ls = u[1], tm = u[2], tls = u[3], qt = v[0], total = v[1], teacher = {v[2], v[3]};
  }
  __device__ __forceinline__ bool dead() const { return m == __uint_as_float(0x7F800000u); }
  __device__ __forceinline__ float p(float x, float c) const { return __builtin_amdgcn_exp2f(fmaf(x - m, c, -ls)); }
  // log2 of the other classes' share
  __device__ __forceinline__ float log2_rest(float c) const { return fmaf(tm - m, c, tls - ls); }
  // derivative of the other classes: coefficient() 2^((x - base()) c - base_log())
  __device__ __forceinline__ bool rest() const { return qt > 0.0f; }
  __device__ __forceinline__ float base() const { return rest() ? tm : m; }
  __device__ __forceinline__ float base_log() const { return rest() ? tls : ls; }
  __device__ __forceinline__ float coefficient(float c) const {
    return rest() ? fmaf(total, __builtin_amdgcn_exp2f(log2_rest(c)), -qt) : total;
  }
  __device__ __forceinline__ void poison() { m = ls = total = qnan(); }
};
__device__ __forceinline__ RowStats dead_row() { return {__uint_as_float(0x7F800000u), 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, {0.0f, 0.0f}}; }

// loss of a row from its sums: cross = sum q (log q - log p), mass = sum q; rest: the classes that are not the teacher's
__device__ __forceinline__ float finish_row(RowStats& st, float cross, float mass, bool with_rest, MaxSum rest, float c) {
  st.qt = st.tm = st.tls = 0.0f;
  st.total = mass;
  if (with_rest && rest.m != ninf()) {
    st.tm = rest.m;
    st.tls = log2_sum(rest);
    st.qt = fmaxf(0.0f, 1.0f - mass);
    if (st.qt > 0.0f) cross += st.qt * (__builtin_amdgcn_logf(st.qt) - st.log2_rest(c)) * kLn2;
    st.total = mass + st.qt;
  }
  return cross;
}

// Marks the teacher's classes of a short row in a bit map of LDS (one bit a class, WORDS words a row); true for the one
// that finds its class marked already.  A wave's LDS operations run in order, so that no barrier is needed within it.
template <int L, int WORDS>
__device__ __forceinline__ void clear_marks(unsigned* marks, int lane) {
  __builtin_amdgcn_wave_barrier();
  for (int w = lane; w < WORDS; w += L) marks[w] = 0u;
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ bool mark(unsigned* marks, int at) {
  const unsigned bit = 1u << (at & 31);
  return atomicOr(&marks[at >> 5], bit) & bit;
}

// What a group of L lanes holds of a short row: NV vectors each, and lane j the teacher's entry j (further ones are read
// when their turn comes).  All of it is asked for at once, a turn of the loop ahead: a row is little work, and one that
// waited for its weight before its logits, and for those before the next row, would spend its time on latency (measured
// at 1474560 rows of 128: 250 us where the traffic takes 80).
template <typename T, int L, int NV>
struct ShortRow {
  u32x4 x[NV];
  float weight = 0.0f, lse = 0.0f, value = 0.0f, g = 0.0f;
  int at = -1;
  RowStats st;
  template <bool GRAD>
  __device__ __forceinline__ void load(const DistillArgs& a, int64_t row, int lane) {
    if (row >= a.rows) {  // whole groups: the row stays unwritten
#pragma unroll
      for (int v = 0; v < NV; ++v) x[v] = u32x4{0u, 0u, 0u, 0u};
      weight = 0.0f;
      return;
    }
    const T* p = (const T*)a.logits + row * a.stride;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (v * L + lane) * Vec<T>::E;
      x[v] = load_row(p, i, i < a.V ? a.V : i);
    }
    weight = a.weights ? a.weights[row] : 1.0f;
    at = lane < a.k ? teacher_index(a, row * a.k + lane) : -1;
    value = lane < a.k ? teacher_value(a, row * a.k + lane) : ninf();
    if (GRAD) {
      st.load(a, row);
      g = a.g_loss[a.reduction == VSL_REDUCE_NONE ? row : 0];
    } else if (a.lse) {
      lse = a.lse[row];
    }
  }
  // f(entry, class or -1, value) for the lane's entries of the teacher
  template <typename F>
  __device__ __forceinline__ void each(const DistillArgs& a, int64_t row, int lane, int k, F f) const {
    if (lane < k) f(lane, at, value);
    for (int j = lane + L; j < k; j += L) f(j, teacher_index(a, row * a.k + j), teacher_value(a, row * a.k + j));
  }
};
constexpr int kResident = 2048;  // blocks of 256 threads that 256 CUs hold: what walks short rows

// Forward pass of short rows: maximum, the teacher's entries from an LDS line, then the sum over all classes or, with a rest
// class, over those that are not the teacher's.  1474560 x 128 bfloat16, k = 8, rest class: 146 us, 3.4 TB/s; bound by
// vector instructions (78 % busy), the exponentials and the two-float logarithms of q.

template <typename T, int L, int NV>
__global__ __launch_bounds__(kThreads) void k_distill_rows(DistillArgs a) {
  constexpr int E = Vec<T>::E, G = kThreads / L, W = L * NV * E;
  __shared__ unsigned marks_of[G][W / 32];
  __shared__ __attribute__((aligned(16))) T lines[G][W];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  unsigned* marks = marks_of[group];
  T* line = lines[group];
  const unsigned long long members = (~0ull >> (64 - L)) << (((threadIdx.x & 63) / L) * L);
  const int64_t step = (int64_t)gridDim.x * G;
  double total = 0.0, count = 0.0;
  ShortRow<T, L, NV> next;
  next.template load<false>(a, (int64_t)blockIdx.x * G + group, lane);
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + group;
    const ShortRow<T, L, NV> in = next;
    if (r0 + step < a.rows) next.template load<false>(a, row + step, lane);
    const bool skip = in.weight == 0.0f;  // the lanes of a group agree
    const int k = skip ? 0 : a.k;
    float xs[NV][E];
    MaxSum all{ninf(), 0.0f}, rest{ninf(), 0.0f};
    clear_marks<L, W / 32>(marks, lane);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      *(u32x4*)(line + (v * L + lane) * E) = in.x[v];
      unpack(in.x[v], xs[v], (const T*)nullptr);
#pragma unroll
      for (int e = 0; e < E; ++e) all.m = __builtin_elementwise_maximum(all.m, xs[v][e]);
    }
    __builtin_amdgcn_wave_barrier();
    TeacherSum teacher{in.lse, kWhole};
    if (!a.lse) {
      MaxSum t{ninf(), 0.0f};
      in.each(a, row, lane, k, [&](int, int, float v) { t.m = __builtin_elementwise_maximum(t.m, v); });
      t.m = group_all<L>(t.m, MaxF());
      const float ref = exp_ref(t.m);
      in.each(a, row, lane, k, [&](int, int, float v) { t.s += exp_of(v, ref, a.c); });
      t.s = group_all<L>(t.s, AddF());
      teacher = {t.m, log2_sum(t) * kLn2};
    }
    all.m = group_all<L>(all.m, MaxF());
    const float ref = exp_ref(all.m);
    bool bad = false, twice = false;
    float mass = 0.0f, cross = 0.0f, seen = 0.0f;
    in.each(a, row, lane, k, [&](int, int at, float v) {
      const LogQ lq = log_q(a, v, teacher);
      const float q = lq.q();
      mass += q;
      bad |= at < 0;
      if (at < 0) return;
      const float z = (float)line[at] - ref;
      if (q != 0.0f) cross += q * (lq.log() - z * a.ih);
      if (mark(marks, at)) twice = true;
      else seen += __builtin_amdgcn_exp2f(z * a.c);  // a class counts once
    });
    bad = (__ballot(bad) & members) != 0;
    if (__ballot(twice) & members) {  // which entry came first is not the hardware's to say: the first in the teacher's order
      seen = 0.0f;
      in.each(a, row, lane, k, [&](int j, int at, float) {
        bool first = at >= 0;
        for (int u = 0; u < j && first; ++u) first = teacher_index(a, row * a.k + u) != at;
        if (first) seen += exp_of((float)line[at], ref, a.c);
      });
    }
    __builtin_amdgcn_wave_barrier();
    if (a.lse) {  // the other classes alone: the teacher's become -infinity in the line, which is read again
      in.each(a, row, lane, k, [&](int, int at, float) {
        if (at >= 0) line[at] = (T)ninf();
      });
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int v = 0; v < NV; ++v) unpack(*(const u32x4*)(line + (v * L + lane) * E), xs[v], (const T*)nullptr);
    }
    auto sum_from = [&](float base) {
      const Exponent ex(base, a.c);
      float s = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          s += ex(xs[v][e]);
          s2 += ex(xs[v][e + 1]);
        }
      return group_all<L>(s + s2, AddF()) * ex.factor();
    };
    const float s = sum_from(ref);
    if (a.lse) {
      all.s = group_all<L>(seen, AddF()) + s;
      rest = {s == 0.0f ? ninf() : all.m, s};
      if (__any(s < 1e-20f)) {  // far below the teacher's classes: their sum from their own maximum, in the rows concerned
        float m = ninf();
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int e = 0; e < E; ++e) m = __builtin_elementwise_maximum(m, xs[v][e]);
        m = group_all<L>(m, MaxF());
        const float own = sum_from(exp_ref(m));
        if (s < 1e-20f) rest = {m, own};  // the row's bits do not depend on the rows that share its wave
      }
    } else {
      all.s = s;
    }
    cross = group_all<L>(cross, AddF());
    mass = group_all<L>(mass, AddF());
    RowStats st;
    st.m = all.m;
    st.ls = log2_sum(all);
    st.teacher = teacher;
    float loss = finish_row(st, cross + mass * (st.ls * kLn2), mass, a.lse != nullptr, rest, a.c) * a.temperature *
                 a.temperature * in.weight;
    if (st.ls != st.ls) st.poison();  // NaN or +infinity among the logits
    if (skip || teacher.base == ninf() || st.m == ninf()) {
      st = dead_row();
      loss = 0.0f;
    }
    if (bad) {
      st.poison();
      loss = qnan();
    }
    if (row < a.rows && lane == 0) {
      st.store(a, row);
      if (a.sums) {
        total += (double)loss;
        count += (double)in.weight;
      } else {
        a.row_loss[row] = loss;
      }
    }
  }
  if (!a.sums) return;
  __shared__ double red[2 * kWaves];
  block_sum2<kWaves>(total, count, red);
  if (threadIdx.x == 0) {
    a.sums[2 * blockIdx.x] = total;
    a.sums[2 * blockIdx.x + 1] = count;
  }
}

// The gradient of a short row: every class as if it were not the teacher's goes to an LDS line, the teacher's entries
// overwrite theirs there, and the line goes out.  1474560 x 128 bfloat16, k = 8: 165 us, 5.3 TB/s read and written.
template <typename T, int L, int NV>
__global__ __launch_bounds__(kThreads) void k_distill_rows_grad(DistillArgs a) {
  constexpr int E = Vec<T>::E, G = kThreads / L, W = L * NV * E;
  __shared__ unsigned marks_of[G][W / 32];
  __shared__ __attribute__((aligned(16))) T lines[G][W];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  unsigned* marks = marks_of[group];
  T* line = lines[group];
  const unsigned long long members = (~0ull >> (64 - L)) << (((threadIdx.x & 63) / L) * L);
  const int64_t step = (int64_t)gridDim.x * G;
  const float divisor = a.reduction == VSL_REDUCE_MEAN ? *a.divisor : 1.0f;
  ShortRow<T, L, NV> next;
  next.template load<true>(a, (int64_t)blockIdx.x * G + group, lane);
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + group;
    const ShortRow<T, L, NV> in = next;
    if (r0 + step < a.rows) next.template load<true>(a, row + step, lane);
    if (row >= a.rows) continue;  // whole groups; what follows is per group
    const RowStats& st = in.st;
    const bool skip = in.weight == 0.0f || st.dead();
    const float g = skip || divisor == 0.0f ? 0.0f : in.g / divisor * in.weight * a.temperature;
    const Exponent ex(st.base(), a.c);
    const float co = g * st.coefficient(a.c) * ex.factor(st.base_log());
    clear_marks<L, W / 32>(marks, lane);
#pragma unroll
    for (int v = 0; v < NV; ++v) *(u32x4*)(line + (v * L + lane) * E) = in.x[v];
    __builtin_amdgcn_wave_barrier();
    // the lane's first entry, kept until the line has become the gradient's
    const float own = lane < a.k && in.at >= 0 ? (float)line[in.at] : 0.0f;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float d[E];
      unpack(in.x[v], d, (const T*)nullptr);
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = co * ex(d[e]);
      if (skip) {
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = 0.0f;
      }
      *(u32x4*)(line + (v * L + lane) * E) = pack(d, (const T*)nullptr);
    }
    __builtin_amdgcn_wave_barrier();
    if (!skip) {
      const T* x = (const T*)a.logits + row * a.stride;
      bool twice = false;
      in.each(a, row, lane, a.k, [&](int j, int at, float v) {
        if (at < 0) return;
        twice |= mark(marks, at);
        const float z = j < L ? own : (float)x[at];
        line[at] = (T)(g * fmaf(st.total, st.p(z, a.c), -log_q(a, v, st.teacher).q()));
      });
      if (__ballot(twice) & members)  // an index occurs twice: every entry takes the sum of its class, in the teacher's order
        in.each(a, row, lane, a.k, [&](int, int at, float) {
          if (at < 0) return;
          float q = 0.0f;
          for (int u = 0; u < a.k; ++u)
            if (teacher_index(a, row * a.k + u) == at) q += log_q(a, teacher_value(a, row * a.k + u), st.teacher).q();
          line[at] = (T)(g * fmaf(st.total, st.p((float)x[at], a.c), -q));
        });
    }
    __builtin_amdgcn_wave_barrier();
    T* out = (T*)a.grad + row * a.grad_stride;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (v * L + lane) * E;
      if (i + E <= a.V) {
        store16(out + i, *(const u32x4*)(line + i));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (i + e < a.V) out[i + e] = line[i + e];
      }
    }
  }
}

// Closes a long row: the first k threads hold the teacher's entries.  `rest`: sums over the classes that are not the
// teacher's when there is a rest class, over all classes otherwise.
template <typename T>
__device__ __forceinline__ void close_row(const DistillArgs& a, int64_t row, float w, MaxSum rest, int* index, float* red) {
  const int tid = threadIdx.x;
  const T* x = (const T*)a.logits + row * a.stride;
  const bool mine = tid < a.k;
  const float value = mine ? teacher_value(a, row * a.k + tid) : ninf();
  const int at = mine ? teacher_index(a, row * a.k + tid) : 0;
  if (mine) index[tid] = at;
  TeacherSum teacher;
  if (a.lse) {
    teacher = {a.lse[row], kWhole};
  } else {
    const MaxSum t = block_join<kWaves>({value, value == ninf() ? 0.0f : 1.0f}, red, a.c);
    teacher = {t.m, log2_sum(t) * kLn2};
  }
  const bool bad = __syncthreads_or(mine && at < 0);
  bool first = mine && at >= 0;
  for (int j = 0; j < tid && first; ++j) first = index[j] != at;
  const float z = mine && at >= 0 ? (float)x[at] : ninf();
  MaxSum all = rest;
  if (a.lse) {
    const MaxSum seen = block_join<kWaves>({first ? z : ninf(), first && z != ninf() ? 1.0f : 0.0f}, red, a.c);
    all = join(rest, seen, a.c);
  }
  RowStats st;
  st.m = all.m;
  st.ls = log2_sum(all);
  st.teacher = teacher;
  const LogQ lq = log_q(a, value, teacher);
  const float q = mine ? lq.q() : 0.0f;
  const float log_p = (z - all.m) * a.ih - st.ls * kLn2;
  const float cross = block_add<kWaves>(q != 0.0f ? q * (lq.log() - log_p) : 0.0f, red);
  const float mass = block_add<kWaves>(q, red);
  float loss = finish_row(st, cross, mass, a.lse != nullptr, rest, a.c) * a.temperature * a.temperature * w;
  if (st.ls != st.ls) st.poison();  // NaN or +infinity among the logits
  if (teacher.base == ninf() || st.m == ninf()) {
    st = dead_row();
    loss = 0.0f;
  }
  if (bad) {
    st.poison();
    loss = qnan();
  }
  if (tid == 0) {
    st.store(a, row);
    a.row_loss[row] = loss;
  }
}

constexpr int kMaxSegment = 1 << 17;  // elements of a segment: one bit of LDS each says whether the class is the teacher's

// Forward pass of long rows, a block per row or segment: one read, running maximum and sum per thread; with a rest class
// (REST) the teacher's classes are left out of them by a bit map.  4096 x 131072 bfloat16: 225 us, 4.8 TB/s.
constexpr int kWide = 4;  // vectors a thread has under way
template <typename T, bool REST>
__global__ __launch_bounds__(kThreads) void k_distill_stream(DistillArgs a) {
  constexpr int E = Vec<T>::E, kSpan = kThreads * E * kWide;
  __shared__ unsigned bits[REST ? kMaxSegment / 32 : 1];
  __shared__ int index[VSL_MAX_TOP];
  __shared__ float red[2 * kWaves];
  const int tid = threadIdx.x;
  const int64_t items = a.rows * a.segs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = item / a.segs;
    const int seg = (int)(item % a.segs);
    const float w = a.weights ? a.weights[row] : 1.0f;
    if (w == 0.0f) {  // the whole block agrees
      if (tid == 0 && seg == 0) {
        dead_row().store(a, row);
        a.row_loss[row] = 0.0f;
      }
      continue;
    }
    const T* x = (const T*)a.logits + row * a.stride;
    const int e0 = seg * a.seg_len, e1 = min(a.V, e0 + a.seg_len);
    if (REST) {
      for (int i = tid; i < (e1 - e0 + 31) / 32; i += kThreads) bits[i] = 0u;
      __syncthreads();
      if (tid < a.k) {
        const int at = teacher_index(a, row * a.k + tid);
        if (at >= e0 && at < e1) atomicOr(&bits[(at - e0) >> 5], 1u << ((at - e0) & 31));
      }
      __syncthreads();
    }
    RunSum run;
    u32x4 next[kWide];
    load_group(x, e0, e1, next);
    for (int i0 = e0; i0 < e1; i0 += kSpan) {
      float v[kWide][E];
#pragma unroll
      for (int u = 0; u < kWide; ++u) unpack(next[u], v[u], (const T*)nullptr);
      if (i0 + kSpan < e1) load_group(x, i0 + kSpan, e1, next);
      if (REST) {
#pragma unroll
        for (int u = 0; u < kWide; ++u) {
          const int i = i0 + (u * kThreads + tid) * E;
          if (i >= e1) continue;
          const unsigned own = (bits[(i - e0) >> 5] >> ((i - e0) & 31)) & ((1u << E) - 1);
          if (own)
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (own >> e & 1) v[u][e] = ninf();
        }
      }
      add_group<T>(v, run, a.c);
    }
    const MaxSum t = block_join<kWaves>(run.get(), red, a.c);
    if (a.segs == 1) {
      close_row<T>(a, row, w, t, index, red);
    } else if (tid == 0) {
      a.partial[2 * item] = t.m;
      a.partial[2 * item + 1] = t.s;
    }
    __syncthreads();
  }
}

// Joins a row's segments and closes it: 7 rows of 32 segments 5 us, latency of the chain partials, entries, logits.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_distill_join(DistillArgs a) {
  __shared__ int index[VSL_MAX_TOP];
  __shared__ float red[2 * kWaves];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float w = a.weights ? a.weights[row] : 1.0f;
    if (w != 0.0f) {
      MaxSum t{ninf(), 0.0f};
      for (int s = threadIdx.x; s < a.segs; s += kThreads)
        t = join(t, {a.partial[2 * (row * a.segs + s)], a.partial[2 * (row * a.segs + s) + 1]}, a.c);
      t = block_join<kWaves>(t, red, a.c);
      close_row<T>(a, row, w, t, index, red);
    }
    __syncthreads();
  }
}

// The gradient of a long row: every class as if it were not the teacher's, then, behind a barrier, the teacher's own.
// 4096 x 131072 bfloat16: 425 us, 5.0 TB/s read and written.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_distill_grad(DistillArgs a) {
  constexpr int E = Vec<T>::E, kTile = kThreads * E;
  __shared__ int index[VSL_MAX_TOP];
  __shared__ float share[VSL_MAX_TOP];
  const int tid = threadIdx.x;
  const int64_t items = a.rows * a.segs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = item / a.segs;
    const int seg = (int)(item % a.segs);
    const float w = a.weights ? a.weights[row] : 1.0f;
    RowStats st;
    st.load(a, row);
    const bool skip = w == 0.0f || st.dead();
    const T* x = (const T*)a.logits + row * a.stride;
    T* out = (T*)a.grad + row * a.grad_stride;
    const int e0 = seg * a.seg_len, e1 = min(a.V, e0 + a.seg_len);
    const float g = skip ? 0.0f : row_scale(a, row, w);
    const Exponent ex(st.base(), a.c);
    const float co = g * st.coefficient(a.c) * ex.factor(st.base_log());
    int at = -1;
    if (!skip && tid < a.k) {
      at = teacher_index(a, row * a.k + tid);
      index[tid] = at;
      share[tid] = log_q(a, teacher_value(a, row * a.k + tid), st.teacher).q();
    }
    for (int i0 = e0; i0 < e1; i0 += kTile) {
      const int i = i0 + tid * E;
      if (i >= e1) break;
      float d[E];
      if (skip) {
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = 0.0f;
      } else {
        unpack(load_row(x, i, e1), d, (const T*)nullptr);
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = co * ex(d[e]);
      }
      if (i + E <= e1) {
        store16(out + i, pack(d, (const T*)nullptr));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (i + e < e1) out[i + e] = (T)d[e];
      }
    }
    __syncthreads();
    if (at >= e0 && at < e1) {
      float q = 0.0f;
      for (int j = 0; j < a.k; ++j)
        if (index[j] == at) q += share[j];
      out[at] = (T)(g * fmaf(st.total, st.p((float)x[at], a.c), -q));  // entries of one index write the same value
    }
    __syncthreads();
  }
}

int check_distill(const vsl_distill_desc* d) {
  if (!d) return fail(VSL_ERR_INVALID_ARGUMENT, "distill: descriptor is null");
  if (int rc = check_matrix("distill", d->logits, d->rows, d->vocab, d->stride, d->type)) return rc;
  if (d->k < 1 || d->k > VSL_MAX_TOP || d->k > d->vocab)
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill: need 1 <= k <= min(vocab, 256)");
  if (bad_type(d->value_type)) return fail(VSL_ERR_INVALID_ARGUMENT, "distill: unknown type of the teacher's values");
  if (d->index_bytes != 4 && d->index_bytes != 8)
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill: teacher indices must be int32 or int64");
  if (d->reduction < VSL_REDUCE_NONE || d->reduction > VSL_REDUCE_MEAN)
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill: unknown reduction");
  if (!(d->temperature >= 1e-4f && d->temperature <= 1e4f))
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill: temperature must lie in 1e-4..1e4");
  if (d->rows > 0 && (!d->logits || !d->teacher_values || !d->teacher_indices))
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill: NULL tensor");
  return VSL_OK;
}

Split distill_split(const vsl_distill_desc* d) {
  if (d->vocab <= short_row(d->type)) return {1, (int)d->vocab};
  const int tile = kThreads * vec_of(d->type);
  Split s = split_row(d->rows, d->vocab, tile, 1, 1 << 20);
  if (s.seg_len > kMaxSegment) {
    s.seg_len = kMaxSegment;
    s.segs = (int)ceil_div(d->vocab, kMaxSegment);
  }
  return s;
}

DistillArgs distill_args(const vsl_distill_desc* d) {
  DistillArgs a{};
  const Split sp = distill_split(d);
  a.logits = d->logits;
  a.values = d->teacher_values;
  a.indices = d->teacher_indices;
  a.lse = d->teacher_lse;
  a.weights = d->weights;
  a.rows = d->rows;
  a.stride = d->stride;
  a.V = (int)d->vocab;
  a.k = d->k;
  a.segs = sp.segs;
  a.seg_len = sp.seg_len;
  a.value_type = d->value_type;
  a.index_bytes = d->index_bytes;
  a.reduction = d->reduction;
  const double inv = 1.0 / (double)d->temperature;
  a.c = (float)(inv * 1.4426950408889634);
  a.ih = (float)inv;
  a.il = (float)(inv - (double)a.ih);
  a.temperature = d->temperature;
  return a;
}

template <typename T, bool GRAD>
int launch_distill(const DistillArgs& a, hipStream_t s) {  // returns the blocks
  const dim3 b(kThreads);
  if (a.V <= 256 * Vec<T>::E) {
    const int nv = (int)ceil_div(a.V, Vec<T>::E);
    auto launch = [&](auto fwd, auto bwd, int lanes) {
      const int64_t blocks = ceil_div(a.rows, kThreads / lanes);
      const dim3 g((unsigned)(blocks < kResident ? blocks : kResident));
      if (GRAD) hipLaunchKernelGGL(bwd, g, b, 0, s, a);
      else hipLaunchKernelGGL(fwd, g, b, 0, s, a);
      return (int)g.x;
    };
    // Fewer lanes a row share the work that every row costs among more rows: 8 lanes of two vectors against 16 of one, 128
    // bins in bfloat16, 146 against 232 us forward.
    if (nv <= 8) return launch(k_distill_rows<T, 8, 1>, k_distill_rows_grad<T, 8, 1>, 8);
    if (nv <= 16) return launch(k_distill_rows<T, 8, 2>, k_distill_rows_grad<T, 8, 2>, 8);
    if (nv <= 32) return launch(k_distill_rows<T, 16, 2>, k_distill_rows_grad<T, 16, 2>, 16);
    if (nv <= 64) return launch(k_distill_rows<T, 16, 4>, k_distill_rows_grad<T, 16, 4>, 16);
    if (nv <= 128) return launch(k_distill_rows<T, 64, 2>, k_distill_rows_grad<T, 64, 2>, 64);
    return launch(k_distill_rows<T, 64, 4>, k_distill_rows_grad<T, 64, 4>, 64);
  }
  const dim3 g(grid_of(a.rows * a.segs));
  if (GRAD) {
    hipLaunchKernelGGL(k_distill_grad<T>, g, b, 0, s, a);
    return (int)g.x;
  }
  if (a.lse) hipLaunchKernelGGL((k_distill_stream<T, true>), g, b, 0, s, a);
  else hipLaunchKernelGGL((k_distill_stream<T, false>), g, b, 0, s, a);
  if (a.segs > 1) hipLaunchKernelGGL(k_distill_join<T>, dim3(grid_of(a.rows)), b, 0, s, a);
  return (int)g.x;
}

int check_workspace(const char* what, const void* workspace, size_t have, size_t need) {
  if (have < need) return fail(VSL_ERR_WORKSPACE_TOO_SMALL, std::string(what) + ": workspace too small");
  if (need && (!workspace || (uintptr_t)workspace % 256))
    return fail(VSL_ERR_INVALID_ARGUMENT, std::string(what) + ": workspace must be 256-byte aligned and not NULL");
  return VSL_OK;
}

}  // namespace
}  // namespace vsl_vocab

using namespace vsl_vocab;

extern "C" {

size_t vsl_top_logits_workspace_bytes(const vsl_top_desc* d) {
  if (check_top(d)) return 0;
  const Split sp = top_split(d);
  if (sp.segs == 1) return 0;
  return up256((size_t)d->rows * sp.segs * d->k * 8) + up256((size_t)d->rows * sp.segs * 8);
}

int vsl_top_logits(const vsl_top_desc* d, void* values, int32_t* indices, float* lse, void* workspace, size_t workspace_bytes,
                   void* stream) {
  if (int rc = check_top(d)) return rc;
  if (d->rows == 0) return VSL_OK;
  if (!d->logits || !values || !indices) return fail(VSL_ERR_INVALID_ARGUMENT, "top_logits: NULL tensor");
  if ((uintptr_t)values % size_of(d->type) || (uintptr_t)indices % 4 || (uintptr_t)lse % 4)
    return fail(VSL_ERR_INVALID_ARGUMENT, "top_logits: misaligned output");
  if (int rc = check_workspace("top_logits", workspace, workspace_bytes, vsl_top_logits_workspace_bytes(d))) return rc;
  const Split sp = top_split(d);
  TopArgs a{};
  a.logits = d->logits;
  a.values = values;
  a.indices = indices;
  a.lse = lse;
  a.keys = (unsigned long long*)workspace;
  a.stat = (float*)((char*)workspace + up256((size_t)d->rows * sp.segs * d->k * 8));
  a.rows = d->rows;
  a.stride = d->stride;
  a.V = (int)d->vocab;
  a.k = d->k;
  a.segs = sp.segs;
  a.seg_len = sp.seg_len;
  a.c = (float)(1.4426950408889634 / (double)d->temperature);
  a.inv_t = (float)(1.0 / (double)d->temperature);
  const bool rows_program = d->vocab <= short_row(d->type);
  hipStream_t s = (hipStream_t)stream;
  if (d->type == VSL_TYPE_F32) launch_top<float>(a, rows_program, s);
  else if (d->type == VSL_TYPE_BF16) launch_top<__bf16>(a, rows_program, s);
  else launch_top<_Float16>(a, rows_program, s);
  return launch_status("top_logits");
}

size_t vsl_distill_workspace_bytes(const vsl_distill_desc* d) {
  if (!d || d->rows < 0 || d->vocab < 1 || bad_type(d->type)) return 0;
  const Split sp = distill_split(d);
  if (d->vocab <= short_row(d->type)) return up256(kResident * 2 * sizeof(double));
  return (sp.segs > 1 ? up256((size_t)d->rows * sp.segs * 8) : 0) + sum_workspace_bytes(d->rows);
}

int vsl_distill_fwd(const vsl_distill_desc* d, float* row_loss, float* loss, float* divisor, float* stats, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (int rc = check_distill(d)) return rc;
  if (d->reduction != VSL_REDUCE_NONE && (!loss || !divisor)) return fail(VSL_ERR_INVALID_ARGUMENT, "distill: NULL loss");
  if (d->rows > 0 && (!row_loss || !stats)) return fail(VSL_ERR_INVALID_ARGUMENT, "distill: NULL output");
  if ((uintptr_t)stats % 16) return fail(VSL_ERR_INVALID_ARGUMENT, "distill: stats must be 16-byte aligned");
  if (int rc = check_workspace("distill", workspace, workspace_bytes, vsl_distill_workspace_bytes(d))) return rc;
  hipStream_t s = (hipStream_t)stream;
  DistillArgs a = distill_args(d);
  a.row_loss = row_loss;
  a.stats = stats;
  const bool reduce = d->reduction != VSL_REDUCE_NONE, short_rows = d->vocab <= short_row(d->type);
  const size_t part = a.segs > 1 ? up256((size_t)d->rows * a.segs * 8) : 0;
  a.partial = (float*)workspace;
  a.sums = reduce && short_rows ? (double*)workspace : nullptr;
  int blocks = 0;
  if (d->rows > 0)
    blocks = d->type == VSL_TYPE_F32 ? launch_distill<float, false>(a, s)
             : d->type == VSL_TYPE_BF16 ? launch_distill<__bf16, false>(a, s) : launch_distill<_Float16, false>(a, s);
  if (reduce && short_rows) launch_sum_pairs(a.sums, blocks, d->reduction, loss, divisor, s);
  else if (reduce) launch_sum(row_loss, d->weights, d->rows, d->reduction, (char*)workspace + part, loss, divisor, s);
  return launch_status("distill");
}

int vsl_distill_bwd(const vsl_distill_desc* d, const float* stats, const float* divisor, const float* g_loss, void* grad,
                    int64_t grad_stride, void* stream) {
  if (int rc = check_distill(d)) return rc;
  if (d->rows == 0) return VSL_OK;
  if (!stats || !g_loss || !grad || (d->reduction == VSL_REDUCE_MEAN && !divisor))
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill backward: NULL tensor");
  if ((uintptr_t)stats % 16 || (uintptr_t)grad % size_of(d->type))
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill backward: misaligned stats or gradient");
  if (grad_stride < d->vocab || grad_stride >= (1LL << 40))
    return fail(VSL_ERR_INVALID_ARGUMENT, "distill backward: the gradient's row stride must be at least vocab");
  DistillArgs a = distill_args(d);
  a.stats = (float*)stats;
  a.divisor = divisor;
  a.g_loss = g_loss;
  a.grad = grad;
  a.grad_stride = grad_stride;
  hipStream_t s = (hipStream_t)stream;
  if (d->type == VSL_TYPE_F32) launch_distill<float, true>(a, s);
  else if (d->type == VSL_TYPE_BF16) launch_distill<__bf16, true>(a, s);
  else launch_distill<_Float16, true>(a, s);
  return launch_status("distill backward");
}

}  // extern "C"
