// Learning from a teacher's top logits.
//
// top_logits_k: the k largest of a row, in the order of (value, lowest index first); a NaN is the
// largest value, as in a sort.  A key of 64 bits (the value's bits made monotone, the index's
// complement) makes all elements of a row distinct, so the answer is the k largest keys.
//
// distill_*: for a row z of V student logits and k named classes c_j with teacher logits t_j
//   p_j = exp(t_j / T - norm), norm = the teacher's lse, or log sum over the named t_j / T
//   q = softmax(z / T), qt = softmax(z / T) within the classes that are not named
//   KD = sum_j p_j (log p_j - log q_{c_j}) [+ r (log r - log sum of q outside), r = 1 - sum_j p_j]
//   loss = (1 - h) T^2 KD + h (-log softmax(z)_y)
//   dz_i = (1 - h) T (S q_i - sum_{j: c_j = i} p_j [- r qt_i outside]) + h (softmax(z)_i - [i = y])
// The bracketed terms belong to a given teacher lse; S = sum_j p_j [+ r].  The classes outside keep a maximum and a sum of
// their own, so what they hold is never the difference of two near numbers, and a row's exponentials
// are taken relative to that maximum: none of them overflows.
#include <algorithm>
#include <type_traits>

#include "lowp.h"
#include "ops.h"

namespace mx {
namespace {

constexpr float kLowest = -3.402823466e+38f;  // start of a running maximum: finite, so -inf - m is -inf
constexpr double kLog2e = 1.4426950408889634;

// monotone bits of a value: NaN above +inf, -0 equal to +0
__device__ __forceinline__ uint32_t order_bits(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float v, uint32_t i) {
  return ((uint64_t)order_bits(v) << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// v_exp_f32 alone: results below 2^-126 are 0
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// running (maximum, sum of exp2((z - m) c))
struct MaxSum {
  float m = kLowest, s = 0.f;
  __device__ __forceinline__ void raise(float z, float c) {
    if (z > m) {
      s *= exp2_raw((m - z) * c);
      m = z;
    }
  }
  __device__ __forceinline__ void add(float z, float c) {
    raise(z, c);
    s += exp2_raw((z - m) * c);
  }
  __device__ __forceinline__ void merge(float om, float os, float c) {
    const float n = fmaxf(m, om);
    s = s * exp2_raw((m - n) * c) + os * exp2_raw((om - n) * c);
    m = n;
  }
};

constexpr int kT = 256;
constexpr int kU = 4;  // pieces of 16 bytes a thread holds: a tile is TB * kU pieces

// 16 bytes at any address.  The forward and the top logits read past the caches: a row is not read again
// soon (2048 x 65536 in bf16: 55 us with it, 60 without).
typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(1)));

// a thread's pieces of the tile at `base` (rows end at `end`); inside the row no lane looks at the end
template <class T, int TB, bool PAST = true>
__device__ __forceinline__ void load_tile(Piece<T>* x, const typename T::store_t* z, int base, int end) {
  constexpr int N = Piece<T>::kN;
  if (base + TB * kU * N <= end) {
    const typename T::store_t* p = z + base + threadIdx.x * N;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const any16* q = reinterpret_cast<const any16*>(p + u * TB * N);
      const any16 b = PAST ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[u].v[j] = b[j];
    }
  } else {
#pragma unroll
    for (int u = 0; u < kU; ++u) x[u].load(z, base + (u * TB + threadIdx.x) * N, end, T::kNegInf);
  }
}

// The running sum of a thread's tiles: exponentials are exp2(z c - R), one fma each, with R the rounded
// m c; `settle` takes the sum to m itself.  A row whose maximum times c leaves fp32 (only masked by a
// type's lowest value, or as large) ends with s = 0 or an infinite R: it is summed again by MaxSum.
struct TileSum {
  float m = kLowest, s = 0.f, R = kLowest;
  __device__ __forceinline__ void raise(float top, float c) {
    if (top > m) {
      m = top;
      const float n = fmaxf(top * c, kLowest);
      s *= exp2_raw(R - n);
      R = n;
    }
  }
  __device__ __forceinline__ float term(float z, float c) const { return exp2_raw(__builtin_fmaf(z, c, -R)); }
  __device__ __forceinline__ float settled(float c) const {
    return s > 0.f ? s * exp2_raw(-__builtin_fmaf(m, c, -R)) : s;
  }
};
__device__ __forceinline__ bool unsettled(float m, double s, float c) { return !(s > 0.f) || !(fabsf(m * c) < INFINITY); }

// over a block of TB threads; every thread gets the result
template <int TB>
__device__ __forceinline__ MaxSum block_merge(MaxSum v, float c, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(v.m, o, 64), os = __shfl_xor(v.s, o, 64);
    v.merge(om, os, c);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[2 * (threadIdx.x >> 6)] = v.m;
    red[2 * (threadIdx.x >> 6) + 1] = v.s;
  }
  __syncthreads();
  MaxSum t;
  for (int w = 0; w < TB / 64; ++w) t.merge(red[2 * w], red[2 * w + 1], c);
  return t;
}

// ---------------------------------------------------------------------------- top logits
// One pass over the row: a block of TB threads takes tiles of TB x kU pieces of 16 bytes into
// registers, and of each piece the maximum and the exponentials' sum.  In the first tile the threshold
// is the largest 16-bit prefix of a value that at least k pieces' maxima reach, so at least k elements
// do, and for independent values hardly more.  A piece that reaches it is noted; in later tiles its
// maximum has to be above the threshold: an equal element comes after k others that are as large.
// When pieces have gathered, their elements become candidates in LDS and the threshold is raised to
// what k of the candidates reach; so a row of V independent values has about k log(V / tile) noted
// pieces.  Where ties overflow the candidates (constant or sorted rows) the k largest keys are selected
// exactly, bit by bit.  In the end a candidate's place is the number of larger keys.
// Bound by the row's bytes; what is done for a noted piece would otherwise be done by a whole wave.  64
// of each of 4096 rows of 131072 in bf16: 233 us, 4.6 TB/s.
//
// Few long rows are split over blocks: each leaves its segment's k largest keys, in order, and its
// sum, and top_merge_k joins them.  50 of one row of 131072 in fp16 over 16 blocks: 9 and 5.5 us, mostly
// barriers one after the other (27 us in one block).
// candidates: twice the largest k and more; a block of one wave has short rows, and many to a CU
constexpr int top_cap(int tb) { return tb == 64 ? 512 : 1024; }
// noted pieces: up to 2 k or 128 stay noted before a tile that may add all of its own
constexpr int top_pieces(int tb) { return 2 * kTopMax + tb * kU; }

struct TopArgs {
  const void* z;
  void* val;
  int32_t* idx;
  float* lse;
  uint64_t* part;  // [rows][nseg][k] keys, 0 behind a segment's last; then [rows][nseg] (m, s)
  int64_t ldz, rows;
  int V, k, nseg, seglen;
  float c, inv_t;
};

// The largest 16-bit prefix p that at least k of a block's values reach, 0 if there are fewer values.
// Two bits a round: count(trial) is a wave's number of values whose prefix is >= trial; the three
// counts of a round (each below 2^20) share a word.  `slots` holds two rounds, so one barrier a round
// is enough.
template <int TB, class F>
__device__ __forceinline__ uint32_t prefix_of(int k, uint64_t* slots, F count) {
  uint32_t p = 0;
#pragma unroll 1
  for (int bit = 14; bit >= 0; bit -= 2) {
    uint64_t c = 0;
#pragma unroll
    for (uint32_t i = 1; i < 4; ++i) c |= (uint64_t)count(p | i << bit) << (20 * (i - 1));
    if constexpr (TB > 64) {
      uint64_t* s = slots + (bit >> 1 & 1) * (TB / 64);
      if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int w = 0; w < TB / 64; ++w) c += s[w];
    }
    const uint32_t m = (1u << 20) - 1;
    const uint32_t i = (int)(c >> 40 & m) >= k ? 3 : (int)(c >> 20 & m) >= k ? 2 : (int)(c & m) >= k ? 1 : 0;
    p |= i << bit;
  }
  return p;
}
__device__ __forceinline__ int wave_count(bool b) { return __popcll(__ballot(b)); }
// a block's total of its waves' counts.  `slots` holds two rounds, so one barrier a round is enough.
template <int TB>
__device__ __forceinline__ int block_count(int wave_total, int* slots, int round) {
  if constexpr (TB == 64) return wave_total;
  int* s = slots + (round & 1) * (TB / 64);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = wave_total;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int w = 0; w < TB / 64; ++w) n += s[w];
  return n;
}

// the number whose order bits these are (0xffffffff: a NaN)
__device__ __forceinline__ float from_order_bits(uint32_t b) {
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// The k largest of the n keys in `from` and of the elements of np noted pieces go to `to`, in any
// order; returns the smallest of them.  There must be k.  Exact: the key is found bit by bit; the
// pieces are read again for every bit, from the caches.
template <class T, int TB>
__device__ __noinline__ uint64_t select_exact(const uint64_t* from, int n, uint64_t* to,
                                              const typename T::store_t* z, const int* piece, int np, int end, int k,
                                              int* slots, int* cnt) {
  const int tid = threadIdx.x;
  constexpr int N = Piece<T>::kN;
  uint64_t t = 0;
  __syncthreads();
#pragma unroll 1
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t trial = t | 1ull << bit;
    int c = 0;
    for (int i = tid; i < (n + 63) / 64 * 64; i += TB) c += wave_count(i < n && from[i] >= trial);
    for (int p = tid; p < (np + 63) / 64 * 64; p += TB) {
      const int i = p < np ? piece[p] : end;
      Piece<T> x;
      x.load(z, i, end, T::kNegInf);
#pragma unroll
      for (int e = 0; e < N; ++e) c += wave_count(i + e < end && order_key(x.get(e), i + e) >= trial);
    }
    if (block_count<TB>(c, slots, bit) >= k) t = trial;
  }
  if (tid == 0) *cnt = 0;
  __syncthreads();
  for (int i = tid; i < n; i += TB)
    if (from[i] >= t) to[atomicAdd(cnt, 1)] = from[i];
  for (int p = tid; p < np; p += TB)
    for (int i = piece[p], e = 0; e < N && i + e < end; ++e) {
      const uint64_t key = order_key(T::load(z[i + e]), i + e);
      if (key >= t) to[atomicAdd(cnt, 1)] = key;
    }
  __syncthreads();
  return t;
}

// Candidates in LDS: two lists, the current one and its length, and the threshold
template <int TB>
struct Candidates {
  uint64_t* list;
  uint64_t* other;
  uint64_t* wide;
  int* cnt;
  int n;
  float t;             // a further element has to be above it
  uint32_t floor = 0;  // its order bits

  // keep those that reach the largest 16-bit prefix that k of them reach
  __device__ __forceinline__ void raise(int k) {
    const int tid = threadIdx.x;
    const uint32_t prefix = prefix_of<TB>(k, wide, [&](uint32_t trial) {
      int c = 0;
      for (int i = tid; i < (n + 63) / 64 * 64; i += TB) c += wave_count(i < n && (uint32_t)(list[i] >> 48) >= trial);
      return c;
    });
    if (tid == 0) *cnt = 0;
    __syncthreads();
    for (int i = tid; i < n; i += TB)
      if ((uint32_t)(list[i] >> 48) >= prefix) other[atomicAdd(cnt, 1)] = list[i];
    __syncthreads();
    n = *cnt;
    swap();
    floor = prefix << 16;
    t = from_order_bits(floor);
  }
  __device__ __forceinline__ void swap() {
    uint64_t* l = list;
    list = other;
    other = l;
  }
};

// Each candidate's place, the number of larger keys, to put(place, key).  Eight keys a step, so a step
// waits once for LDS; the list is filled up with zeros, which are below every key.
template <int TB, class F>
__device__ __forceinline__ void rank_all(uint64_t* list, int n, F put) {
  const int tid = threadIdx.x, n8 = (n + 7) / 8 * 8;
  if (n + tid < n8) list[n + tid] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += TB) {
    const uint64_t key = list[i];
    int place = 0;
    for (int j = 0; j < n8; j += 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) place += list[j + e] > key;
    }
    put(place, key);
  }
}

// the row's rank-th answer; the first one's writer has the sum: an infinite or NaN maximum is its value
template <class T>
__device__ __forceinline__ void put_top(const TopArgs& a, int64_t row, int rank, uint64_t key,
                                        const typename T::store_t* z, const MaxSum& ms) {
  const uint32_t at = key_index(key);
  static_cast<typename T::store_t*>(a.val)[row * a.k + rank] = z[at];
  a.idx[row * a.k + rank] = (int32_t)at;
  if (rank == 0) {
    const float v = T::load(z[at]);
    a.lse[row] = v - v == 0.f ? ms.m * a.inv_t + logf(ms.s) : v;
  }
}

template <class T, int TB>
__global__ __launch_bounds__(TB) void top_logits_k(TopArgs a) {
  constexpr int N = Piece<T>::kN, TILE = TB * kU * N, kCap = top_cap(TB);
  static_assert(kCap >= 2 * kTopMax, "a list that was cut to k leaves half of its room");
  __shared__ __attribute__((aligned(16))) uint64_t buf[2][kCap];
  __shared__ int piece[top_pieces(TB)];
  __shared__ int slots[2 * TB / 64], cnt, noted;
  __shared__ uint64_t wide[2 * TB / 64];
  __shared__ float red[2 * TB / 64];
  const int tid = threadIdx.x, k = a.k;
  const int64_t row = blockIdx.x / a.nseg;
  const int seg = blockIdx.x % a.nseg, begin = seg * a.seglen, end = min(a.V, begin + a.seglen);
  const auto* z = static_cast<const typename T::store_t*>(a.z) + row * a.ldz;
  const int gather = max(2 * k, 128);
  Candidates<TB> cand{buf[0], buf[1], wide, &cnt, 0, 0.f};
  TileSum ts;
  if (tid == 0) cnt = noted = 0;
#pragma unroll 1
  for (int base = begin; base < end; base += TILE) {
    Piece<T> x[kU];
    float top[kU], f[kU * N];
    load_tile<T, TB>(x, z, base, end);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
#pragma unroll
      for (int e = 0; e < N; ++e) f[u * N + e] = x[u].get(e);
      top[u] = f[u * N];
#pragma unroll
      for (int e = 1; e < N; ++e) top[u] = fmaxf(top[u], f[u * N + e]);
    }
    ts.raise(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), a.c);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kU * N; ++e) s += ts.term(f[e], a.c);
    ts.s += s;
    const bool odd = s != s;  // the sum is NaN: there may be one, or infinities
    // the largest prefix that k of the tile's maxima reach (a piece of NaN alone counts as one)
    auto tile_prefix = [&] {
      uint32_t key[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        key[u] = base + (u * TB + tid) * N < end ? order_bits(top[u]) >> 16 : 0;
      return prefix_of<TB>(k, wide, [&](uint32_t trial) {
               int c = 0;
#pragma unroll
               for (int u = 0; u < kU; ++u) c += wave_count(key[u] >= trial);
               return c;
             }) << 16;
    };
    const bool first = base == begin;
    const int before = noted;
    if (first) {
      cand.floor = tile_prefix();
      cand.t = from_order_bits(cand.floor);
    }
    __syncthreads();  // every thread has `before`
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i0 = base + (u * TB + tid) * N;
      if (i0 < end && (odd || (first ? order_bits(top[u]) >= cand.floor : top[u] > cand.t)))
        piece[atomicAdd(&noted, 1)] = i0;
    }
    __syncthreads();
    const int np = noted;
    __syncthreads();  // every thread has it: what follows is block-uniform
    const bool last = base + TILE >= end;
    if (np > gather || last) {
      // most of the tile above the threshold: a row that rises.  The tile has a threshold of its own.
      if (!first && np - before > TB * kU / 2) cand.floor = max(cand.floor, tile_prefix());
      for (int p = tid; p < np; p += TB) {
        const int i0 = piece[p];
        Piece<T> y;
        y.load(z, i0, end, T::kNegInf);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v = y.get(e);
          if (i0 + e < end && order_bits(v) >= cand.floor) {
            const int pos = atomicAdd(&cnt, 1);
            if (pos < kCap) cand.list[pos] = order_key(v, i0 + e);
          }
        }
      }
      __syncthreads();
      const int had = cand.n;
      cand.n = cnt;
      __syncthreads();  // every thread has read both counters
      cand.t = from_order_bits(cand.floor);
      // the last candidates are ordered: worth it only where there are many
      if (cand.n <= kCap && cand.n > (last ? k + 192 : k + 16)) cand.raise(k);
      if (cand.n > (last ? kCap : kCap / 2)) {
        const bool over = cand.n > kCap;  // the list is what it was before, the rest is in the pieces
        const uint64_t low = select_exact<T, TB>(cand.list, over ? had : cand.n, cand.other, z, piece, over ? np : 0,
                                                 end, k, slots, &cnt);
        cand.floor = (uint32_t)(low >> 32);
        cand.t = from_order_bits(cand.floor);
        cand.swap();
        cand.n = k;
      }
      if (tid == 0) noted = 0;
      __syncthreads();
    }
  }
  MaxSum ms;
  ms.m = ts.m;
  ms.s = ts.settled(a.c);
  ms = block_merge<TB>(ms, a.c, red);
  if (unsettled(ms.m, ms.s, a.c)) {
    ms = MaxSum();
    for (int i = begin + tid; i < end; i += TB) ms.add(T::load(z[i]), a.c);
    ms = block_merge<TB>(ms, a.c, red);
  }
  const int kk = min(k, cand.n);
  rank_all<TB>(cand.list, cand.n, [&](int rank, uint64_t key) {
    if (rank >= kk) return;
    if (a.nseg == 1) put_top<T>(a, row, rank, key, z, ms);
    else a.part[(row * a.nseg + seg) * k + rank] = key;
  });
  if (a.nseg > 1) {
    for (int i = kk + tid; i < k; i += TB) a.part[(row * a.nseg + seg) * k + i] = 0;
    if (tid == 0) reinterpret_cast<float2*>(a.part + a.rows * a.nseg * k)[row * a.nseg + seg] = make_float2(ms.m, ms.s);
  }
}

// The k largest of a row's nseg sorted lists of k keys.  As many keys as k reach the smallest of the
// lists' (k / nseg)-th, and the largest of their last: what is below either is out.
template <class T>
__global__ __launch_bounds__(kT) void top_merge_k(TopArgs a) {
  constexpr int kCap = top_cap(kT);
  __shared__ __attribute__((aligned(16))) uint64_t buf[2][kCap];
  __shared__ int slots[2 * kT / 64], cnt;
  __shared__ uint64_t wide[2 * kT / 64];
  __shared__ float red[2 * kT / 64];
  const int tid = threadIdx.x, k = a.k, total = a.nseg * k;
  const int64_t row = blockIdx.x;
  const auto* z = static_cast<const typename T::store_t*>(a.z) + row * a.ldz;
  const uint64_t* keys = a.part + row * total;
  Candidates<kT> cand{buf[0], buf[1], wide, &cnt, 0, 0.f};
  MaxSum ms;
  const int each = (k + a.nseg - 1) / a.nseg, lane = tid & 63;  // nseg <= 32
  uint64_t least = lane < a.nseg ? keys[lane * k + each - 1] : ~0ull, last = lane < a.nseg ? keys[lane * k + k - 1] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t x = __shfl_xor((unsigned long long)least, o, 32), y = __shfl_xor((unsigned long long)last, o, 32);
    least = x < least ? x : least;
    last = y > last ? y : last;
  }
  least = __shfl((unsigned long long)least, 0, 64);
  last = __shfl((unsigned long long)last, 0, 64);
  const uint64_t floor = least > last ? least : last;
  if (tid < a.nseg) {
    const float2 p = reinterpret_cast<const float2*>(a.part + a.rows * total)[row * a.nseg + tid];
    ms.m = p.x;
    ms.s = p.y;
  }
  if (tid == 0) cnt = 0;
  ms = block_merge<kT>(ms, a.c, red);
  for (int i = tid; i < total; i += kT)
    if (keys[i] >= floor && keys[i] != 0) {
      const int pos = atomicAdd(&cnt, 1);
      if (pos < kCap) cand.list[pos] = keys[i];
    }
  __syncthreads();
  cand.n = cnt;
  __syncthreads();
  if (cand.n > kCap) {
    select_exact<T, kT>(keys, total, cand.list, z, nullptr, 0, 0, k, slots, &cnt);
    cand.n = k;
  } else if (cand.n > k + 192) {
    cand.raise(k);
  }
  rank_all<kT>(cand.list, cand.n, [&](int rank, uint64_t key) {
    if (rank < k) put_top<T>(a, row, rank, key, z, ms);
  });
}

// blocks of a row: long rows that alone would not fill the machine are cut into pieces of 8,192
// classes or more, one tile of a block of 256 threads for a 16-bit type
int row_segments(int64_t rows, int V) {
  const int64_t want = (2 * device_cu_count() + rows - 1) / std::max<int64_t>(rows, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, (V + 8191) / 8192, 32}));
}

int segment_length(int V, int* nseg) {
  const int len = *nseg == 1 ? V : (cdiv(V, *nseg) + 63) / 64 * 64;
  *nseg = cdiv(V, len);
  return len;
}

template <class T, int TB>
void launch_top(const TopArgs& a, hipStream_t st) {
  const int64_t blocks = a.rows * a.nseg;
  MX_LAUNCH((top_logits_k<T, TB>), dim3((uint32_t)blocks), dim3(TB), 0, st, a);
}

__device__ __forceinline__ int64_t load_int(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// sums over a block of each of v[0 .. NV - 1]; every thread gets them
template <int NV>
__device__ __forceinline__ void block_sums(double* v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] += __shfl_xor(v[i], o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < NV; ++i) red[NV * (threadIdx.x >> 6) + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = 0;
    for (int w = 0; w < kT / 64; ++w) v[i] += red[NV * w + i];
  }
}
// maxima over a block, NaN left aside
__device__ __forceinline__ float2 block_max2(float2 v, double* red) {
  float2* r = reinterpret_cast<float2*>(red);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v.x = fmaxf(v.x, __shfl_xor(v.x, o, 64));
    v.y = fmaxf(v.y, __shfl_xor(v.y, o, 64));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < kT / 64; ++w) {
    v.x = fmaxf(v.x, r[w].x);
    v.y = fmaxf(v.y, r[w].y);
  }
  return v;
}

// exp(x) - 1 for x <= 0 within a few parts in 2^53 of its size: x = k log 2 + f with |f| <= 0.35, and
// the power series of exp(f) - 1, whose first term left out is below 2^-55 of f
__device__ __forceinline__ double expm1_neg(double x) {
  x = x < -800.0 ? -800.0 : x;  // -1 from there on; a NaN stays one
  const double k = rint(x * kLog2e);
  const double f = __builtin_fma(-k, 2.3190468138462996e-17, __builtin_fma(-k, 0.6931471805599453, x));
  double r = 1.0 / 6227020800.0;
  constexpr double c[12] = {1.0,         1.0 / 2,     1.0 / 6,      1.0 / 24,      1.0 / 120,      1.0 / 720,
                            1.0 / 5040,  1.0 / 40320, 1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600};
#pragma unroll
  for (int i = 11; i >= 0; --i) r = __builtin_fma(r, f, c[i]);
  const double s = ldexp(1.0, (int)k);
  return __builtin_fma(s, r * f, s - 1.0);
}
// x e^x - e^x + 1 = sum x^n (n - 1) / n!, for |x| <= 1/4: the first term left out is below 2^-54 of the sum
__device__ __forceinline__ double gain_near(double x) {
  double r = 0;
  constexpr double c[13] = {1.0 / 2,           2.0 / 6,           3.0 / 24,          4.0 / 120,         5.0 / 720,
                            6.0 / 5040,        7.0 / 40320,       8.0 / 362880,      9.0 / 3628800,     10.0 / 39916800,
                            11.0 / 479001600,  12.0 / 6227020800.0, 13.0 / 87178291200.0};
#pragma unroll
  for (int i = 12; i >= 0; --i) r = __builtin_fma(r, x, c[i]);
  return r * x * x;
}

// what a row's named entries are: class (or -1) and its teacher logit; k <= kT, one entry a thread
__device__ __forceinline__ void load_entry(const DistillArgs& a, int64_t row, int* cls, float* t) {
  *cls = -1;
  *t = 0;
  if ((int)threadIdx.x >= a.k) return;
  const int64_t c = load_int(a.ti, row * a.k + threadIdx.x, a.ti64);
  const float v = load_any(a.tv, row * a.k + threadIdx.x, a.tv_type);
  if (c >= 0 && c < a.V && !(v == -INFINITY)) {
    *cls = (int)c;
    *t = v;
  }
}

// ---------------------------------------------------------------------------- distillation loss
// Forward: a block takes a row, or a segment of one where there are few rows, in pieces of 16 bytes;
// bound by the row's bytes.  Classes outside the named ones are told by a bit each in LDS, looked at
// once a piece.  Backward: the same pieces, read again and written; the named classes and the label
// are written over afterwards by their own threads.  The gradient is not written by the forward: that
// would save a pass only where the loss's own gradient is 1, and cost one (870 us for 600) elsewhere.
// 4096 x 131072 in bf16 with the teacher's normaliser: forward 184 us (a plain read's rate), backward
// 418 us (5.1 TB/s); 1023 x 50001 in fp16: 30 to 35 us and 40 to 47 us (rows of no alignment; 32 and 37 with
// rows of 50048).
//
// T^2 KD is of the logits' size at any T, so KD is of 1 / T^2, and what it is made of must not be
// rounded at 1.  A row's sum of exponentials is held as S = n + e.  Up to T = kNearT n = 0 and e is a sum of
// fp32 exponentials, joined in 64 bits; what they are rounded by reaches the loss T^2 times (a loss of 1
// over 100 classes: 3e-7 at T = 4, 2e-6 at 8).  Above it n counts classes and e sums exp(z / T) - 1 in 64
// bits, itself of 1 / T.  With log S = log n + log1p(e / n), and the teacher's sum the same way,
// d_j = log p_j - log q_j is right to its last bits, and
//   KD = sum_j (p_j d_j - p_j + q_j) + (r log(r / q_out) - r + q_out)
// has no term below 0 and each of the order of d^2, so nothing cancels (without the rest's term what
// p and q do not sum to is added as it is).  The gradients are q_j (exp(d_j) - 1) likewise, at any T.
// Above kNearT the forward is bound by 64-bit arithmetic: 4096 x 131072 in bf16 680 us, 184 below; 4096 x
// 1000 in fp32 47 us and 23.  The fp32 sums at T = 20 would be off by 1e-5, at 100 by 3e-4.
constexpr double kNearT = 8.0;
constexpr int kMaskWords = 4096;  // a thread's elements of a tile have one: 131,072 classes at a time, 65,536 of fp32

// exponentials relative to the maximum m: their sum at T is n + e, at 1 (where the labels need it) s1
struct Sums {
  float m = kLowest;
  double n = 0, e = 0, s1 = 0;
  // relative to another maximum, at or above m
  __device__ __forceinline__ void move(float to, double inv_t) {
    const double d = (double)m - to;
    if (n > 0) e += expm1_neg(d * inv_t) * (n + e);
    else e = e == 0 ? 0.0 : e * exp(d * inv_t);
    s1 = s1 == 0 ? 0.0 : s1 * exp(d);
    m = to;
  }
};

// running sum of a thread's tiles, as TileSum, joined in 64 bits
struct WideSum {
  float m = kLowest, R = kLowest;
  double s = 0;
  __device__ __forceinline__ void raise(float top, float c) {
    if (top > m) {
      m = top;
      const float n = fmaxf(top * c, kLowest);
      s *= exp2_raw(R - n);
      R = n;
    }
  }
  __device__ __forceinline__ float term(float z, float c) const { return exp2_raw(__builtin_fmaf(z, c, -R)); }
  // what R was rounded by is taken back: for a small y, exp(-y) = 1 - y + y^2 / 2 to 2^-28
  __device__ __forceinline__ double settled(float c) const {
    const float x = __builtin_fmaf(m, c, -R);
    const double y = x / kLog2e;
    return !(s > 0) ? s : s * (fabsf(x) < 0x1p-9f ? 1.0 - y * (1.0 - 0.5 * y) : (double)exp2_raw(-x));
  }
};

// classes [begin, end) of a row; `two`: both sums; `masked`: without the named classes.  The mask has a
// word for each thread and tile, with a bit for each of its elements.
template <class T, bool FAR>
__device__ __forceinline__ Sums row_sums(const DistillArgs& a, const typename T::store_t* z, int begin, int end,
                                         int cls, bool two, uint32_t* mask, double* red) {
  constexpr int N = Piece<T>::kN, TILE = kT * kU * N, kMasked = kMaskWords / kT * TILE;
  static_assert(kU * N <= 32, "a word has a bit for each of a thread's elements");
  const int tid = threadIdx.x;
  const float c = (float)(kLog2e / a.temperature), c1 = (float)kLog2e;
  const bool masked = FAR || a.tlse != nullptr;
  auto word = [](int i) { return i / TILE * kT + i / N % kT; };
  auto bit = [](int i) { return i / (kT * N) % kU * N + i % N; };
  auto set_mask = [&](int v0, int n) {
    __syncthreads();
    for (int i = tid; i < (n + TILE - 1) / TILE * kT; i += kT) mask[i] = 0;
    __syncthreads();
    if (cls >= v0 && cls < v0 + n) atomicOr(&mask[word(cls - v0)], 1u << bit(cls - v0));
    __syncthreads();
  };
  // f(a thread's elements of a tile), -inf for the named ones and behind the end
  auto tiles = [&](auto f) {
    for (int v0 = begin; v0 < end; v0 += kMasked) {
      const int n = min(end - v0, kMasked);
      if (masked) set_mask(v0, n);
#pragma unroll 1
      for (int base = 0; base < n; base += TILE) {
        Piece<T> x[kU];
        float v[kU * N];
        load_tile<T, kT, !FAR>(x, z + v0, base, n);
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e) v[u * N + e] = x[u].get(e);
        if (masked) {
          const uint32_t bits = mask[base / TILE * kT + tid];
          if (bits) {
#pragma unroll
            for (int e = 0; e < kU * N; ++e) v[e] = bits >> e & 1 ? -INFINITY : v[e];
          }
        }
        f(v);
      }
    }
  };
  Sums r;
  if constexpr (FAR) {
    // the maximum first (the row is read again, through the caches), then each class's deviation
    float top = kLowest;
    tiles([&](const float* v) {
#pragma unroll
      for (int e = 0; e < kU * N; ++e) top = fmaxf(top, v[e]);
    });
    r.m = block_max2(make_float2(top, kLowest), red).x;
    const double inv_t = 1.0 / a.temperature;
    int n = 0;
    double s[3] = {0, 0, 0};
    tiles([&](const float* v) {
      float s1 = 0.f;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        bool some = false;
#pragma unroll
        for (int e = u * N; e < (u + 1) * N; ++e) some = some || v[e] != -INFINITY;
        if (!__any(some)) continue;  // pieces behind the end of a short row
#pragma unroll
        for (int e = u * N; e < (u + 1) * N; ++e) {
          const bool in = v[e] != -INFINITY;
          const double x = expm1_neg(((double)v[e] - r.m) * inv_t);
          n += in;
          s[1] += in ? x : 0.0;
          if (two) s1 += exp2_raw((v[e] - r.m) * c1);
        }
      }
      s[2] += s1;
    });
    s[0] = n;
    block_sums<3>(s, red);
    r.n = s[0];
    r.e = s[1];
    r.s1 = s[2];
  } else {
    WideSum t, t1;
    tiles([&](const float* v) {
      float top = v[0], s = 0.f;
#pragma unroll
      for (int e = 1; e < kU * N; ++e) top = fmaxf(top, v[e]);
      t.raise(top, c);
#pragma unroll
      for (int e = 0; e < kU * N; ++e) s += t.term(v[e], c);
      t.s += s;
      if (two) {
        float s1 = 0.f;
        t1.raise(top, c1);
#pragma unroll
        for (int e = 0; e < kU * N; ++e) s1 += t1.term(v[e], c1);
        t1.s += s1;
      }
    });
    auto join = [&](float m, double s, double s1) {
      r.m = block_max2(make_float2(m, kLowest), red).x;
      double v[2] = {s * exp2_raw((m - r.m) * c), s1 * exp2_raw((m - r.m) * c1)};
      block_sums<2>(v, red);
      r.e = v[0];
      r.s1 = v[1];
    };
    join(t.m, t.settled(c), two ? t1.settled(c1) : 0.0);
    if (unsettled(r.m, r.e, c) || (two && unsettled(r.m, r.s1, c1))) {
      MaxSum o, o1;
      for (int v0 = begin; v0 < end; v0 += kMasked) {
        const int n = min(end - v0, kMasked);
        if (masked) set_mask(v0, n);
        for (int i = tid; i < n; i += kT) {
          if (masked && (mask[word(i)] >> bit(i) & 1)) continue;
          const float x = T::load(z[v0 + i]);
          o.add(x, c);
          if (two) o1.add(x, c1);
        }
      }
      join(o.m, o.s, two ? o1.s : 0.f);
    }
  }
  return r;
}

struct RowShared {
  double red[4 * kT / 64];
  int cls[kT];
};

// the row's named entry of this thread, the label, whether the row counts (block-wide)
struct RowEntry {
  int cls;
  float t;
  bool any, counted;
  int64_t y;
  __device__ __forceinline__ RowEntry(const DistillArgs& a, int64_t row, RowShared& sh) {
    load_entry(a, row, &cls, &t);
    sh.cls[threadIdx.x] = cls;
    any = __syncthreads_or(cls >= 0);
    y = a.target ? load_int(a.target, row, a.target64) : -1;
    counted = a.target ? y >= 0 && y < a.V : any;
  }
};

// What the backward needs of a row, in its kDistillStats floats.  A class outside the named ones gets
// co exp((z - ref) / T) + h1 exp(z - top).  A named class has q = ci exp((z - top) / T), with the weight
// w = (1 - h) T in it and what p and the rest sum to; an entry of it has p = w exp((t - tref) / T - norm),
// and log(p / q) = ((t - tref) - (z - top)) / T + K.
struct RowStats {
  float ref, co, top, ci, h1, used, tref, unused;
  double norm, K;
};
static_assert(sizeof(RowStats) == kDistillStats * sizeof(float), "a row's statistics");

// the row's loss and what its backward needs, from the sums over the classes outside the named ones
// (FAR, or with the teacher's lse) or over all
template <class T, bool FAR>
__device__ __forceinline__ void finish_row(const DistillArgs& a, int64_t row, const typename T::store_t* z,
                                           const RowEntry& r, Sums out, RowShared& sh, float* loss_rows) {
  const int tid = threadIdx.x;
  const double inv_t = 1.0 / a.temperature;
  const bool tail = a.tlse != nullptr, masked = FAR || tail, two = a.hard > 0 && a.temperature != 1.0;
  const bool mine = r.cls >= 0, has_out = out.n > 0 || out.e > 0 || out.e != out.e;
  const float zc = mine ? T::load(z[r.cls]) : 0.f;
  bool first = mine;  // this entry is its class's first
  if (masked) {
    for (int j = 0; j < a.k; j += 8) {  // threads without an entry hold -1
#pragma unroll
      for (int e = 0; e < 8; ++e) first = first && (j + e >= tid || sh.cls[j + e] != r.cls);
    }
  }
  RowStats st = {};
  const float2 most = block_max2(make_float2(masked && mine ? zc : kLowest, mine ? r.t : kLowest), sh.red);
  st.top = fmaxf(out.m, most.x);
  st.tref = tail || !r.any ? 0.f : most.y;
  // Waves without an entry only meet the others at the sums.  An entry's exponents are dz / T and dt / T.
  const bool busy = (tid & ~63) < a.k;
  const double dz = (double)zc - st.top, dt = (double)r.t - st.tref;
  const bool live = masked && first && zc != -INFINITY;
  double v[4] = {0, 0, 0, 0}, xz = 0;
  if (busy && mine) {
    xz = FAR ? expm1_neg(dz * inv_t) : exp(dz * inv_t);
    if (live) v[0] = xz;
    if (live && two) v[1] = exp(dz);
    if (!tail) v[2] = FAR ? expm1_neg(dt * inv_t) : exp(dt * inv_t);
    // how many classes the entries name and how many entries there are, each at most 256
    if (FAR) v[3] = (live ? 1.0 : 0.0) + 512.0;
  }
  if constexpr (FAR) block_sums<4>(v, sh.red);
  else if (tail) block_sums<2>(v, sh.red);
  else block_sums<1>(v + 2, sh.red);
  const double own = out.n + out.e;  // the sum outside, relative to its own maximum
  const double shift = ((double)out.m - st.top) * inv_t;
  double q_out = 0, S = 0, s1 = 0, whole = 0, part = 0;  // log S = whole + part
  if (busy) {
    const double entries = FAR ? floor(v[3] / 512) : 0.0, in = FAR ? v[3] - 512 * entries : 0.0;
    Sums all = out;
    if (has_out && out.m != st.top) all.move(st.top, inv_t);
    q_out = all.n + all.e;
    all.n += in;
    all.e += v[0];
    s1 = all.s1 + v[1];
    S = all.n + all.e;
    // `whole` cancels where the teacher's sum has as many classes
    if (FAR) whole = log(all.n);
    part = FAR ? log1p(all.e / all.n) : log(S);
    if (tail) {
      st.norm = a.tlse[row];
      st.K = whole + part - st.norm;
    } else if (r.any) {
      const double w0 = FAR ? log(entries) : 0.0, p0 = FAR ? log1p(v[2] / entries) : log(v[2]);
      st.norm = w0 + p0;
      st.K = (whole - w0) + (part - p0);
    }
  }
  v[0] = v[1] = v[2] = v[3] = 0;
  if (busy && mine) {
    const double p = exp(dt * inv_t - st.norm), d = (dt - dz) * inv_t + st.K;
    const double pd = p == 0 ? 0.0 : p * d;  // p = 0 has no term, whatever the student's value
    v[0] = pd;
    v[1] = p;
    if constexpr (FAR) {
      const double q = (1.0 + xz) / S, gain = gain_near(d);
      const bool near = fabs(d) < 0.25;
      v[0] = near ? q * gain : pd - p + q;
      v[2] = near ? q * ((d - gain) / (1.0 - d)) : p - q;  // q (exp(d) - 1)
      v[3] = first ? 0.0 : q;
    }
  }
  if constexpr (FAR) block_sums<4>(v, sh.red);
  else if (tail) block_sums<2>(v, sh.red);
  else block_sums<1>(v, sh.red);
  if (tid != 0) return;
  double kd = v[0], co = 0, mass = 1;  // co exp((z - ref) / T): what a class outside gets
  const double h = a.hard, w = (1 - h) * a.temperature, sum_p = tail ? v[1] : r.any ? 1.0 : 0.0;
  q_out = has_out ? q_out / S : 0.0;
  if (tail && has_out && !(sum_p >= 1)) {
    const double rest = 1 - sum_p, log_q_out = shift + log(own) - whole - part;
    if constexpr (FAR) {
      const double less = v[2] + v[3], x = -less / q_out;  // less = q_out - rest
      kd += fabs(x) < 0.2 ? q_out * gain_near(log1p(x)) : rest * (log(rest) - log_q_out) - rest + q_out;
      kd -= v[3];
      co = less / own;
    } else {
      kd += rest * (log(rest) - log_q_out);
      co = exp(shift) / S - rest / own;
    }
  } else {
    if (FAR) kd += (sum_p - 1) + q_out - v[3];
    mass = sum_p;
    if (tail) st.K -= log(mass);
    co = has_out ? sum_p * exp(shift) / S : S > 0 ? 0.0 : __builtin_nan("");  // a row of -inf has no distribution
  }
  if (!r.any) kd = 0;
  st.ref = has_out ? out.m : st.top;
  // a weight of 0 takes the term out, whatever the teacher says (KD is infinite where a named class is masked)
  const double z1 = two ? s1 : S;
  double loss = w == 0 ? 0.0 : w * a.temperature * kd;
  if (h > 0) loss += h * (log(z1) - ((double)T::load(z[r.y]) - st.top));
  loss_rows[row] = (float)loss;
  st.co = (float)((w == 0 ? 0.0 : w * co) + (h > 0 && !two ? h * exp((double)st.ref - st.top) / z1 : 0.0));
  st.ci = r.any && w != 0 ? (float)(w * mass / S) : 0.f;
  st.h1 = h > 0 ? (float)(h / z1) : 0.f;
  st.used = 1.f;
  reinterpret_cast<RowStats*>(a.stats)[row] = st;
}

__device__ __forceinline__ void leave_out(const DistillArgs& a, int64_t row, float* loss_rows) {
  if (threadIdx.x == 0) loss_rows[row] = 0.f;
  if (threadIdx.x < kDistillStats) a.stats[row * kDistillStats + threadIdx.x] = 0.f;
}

// part == nullptr: a block has the whole row; else [rows][nseg] sums of a segment each, for distill_join_k
template <class T, bool FAR>
__global__ __launch_bounds__(kT, FAR ? 4 : 8) void distill_fwd_k(DistillArgs a, int nseg, int seglen,
                                                                 double* __restrict__ part,
                                                                 float* __restrict__ loss_rows) {
  __shared__ RowShared sh;
  __shared__ uint32_t mask[kMaskWords];
  const int64_t row = blockIdx.x / nseg;
  const int seg = blockIdx.x % nseg;
  const auto* z = static_cast<const typename T::store_t*>(a.z) + row * a.ldz;
  const RowEntry r(a, row, sh);
  if (!r.counted) {
    if (!part) leave_out(a, row, loss_rows);
    return;
  }
  const bool two = a.hard > 0 && a.temperature != 1.0;
  const Sums out = row_sums<T, FAR>(a, z, seg * seglen, min(a.V, (seg + 1) * seglen), r.cls, two, mask, sh.red);
  if (!part) {
    finish_row<T, FAR>(a, row, z, r, out, sh, loss_rows);
  } else if (threadIdx.x == 0) {
    double* p = part + (row * nseg + seg) * 4;
    p[0] = out.m;
    p[1] = out.n;
    p[2] = out.e;
    p[3] = out.s1;
  }
}

template <class T, bool FAR>
__global__ __launch_bounds__(kT) void distill_join_k(DistillArgs a, int nseg, const double* __restrict__ part,
                                                     float* __restrict__ loss_rows) {
  __shared__ RowShared sh;
  const int64_t row = blockIdx.x;
  const auto* z = static_cast<const typename T::store_t*>(a.z) + row * a.ldz;
  const RowEntry r(a, row, sh);
  if (!r.counted) return leave_out(a, row, loss_rows);
  Sums v;
  if ((int)threadIdx.x < nseg) {
    const double* p = part + (row * nseg + threadIdx.x) * 4;
    v.m = (float)p[0];
    v.n = p[1];
    v.e = p[2];
    v.s1 = p[3];
  }
  v.move(block_max2(make_float2(v.m, kLowest), sh.red).x, 1.0 / a.temperature);
  double s[3] = {v.n, v.e, v.s1};
  block_sums<3>(s, sh.red);
  v.n = s[0];
  v.e = s[1];
  v.s1 = s[2];
  finish_row<T, FAR>(a, row, z, r, v, sh, loss_rows);
}

// loss = the sum or mean of the rows' losses; the rows' weight goes behind their statistics
__global__ __launch_bounds__(1024) void distill_mean_k(const float* __restrict__ loss_rows, float* __restrict__ stats,
                                                       int64_t rows, int mean, float* __restrict__ loss) {
  __shared__ double red[2][16];
  double s = 0, n = 0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    s += loss_rows[i];
    n += reinterpret_cast<const RowStats*>(stats)[i].used;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = s;
    red[1][threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = n = 0;
    for (int w = 0; w < 16; ++w) {
      s += red[0][w];
      n += red[1][w];
    }
    const double inv = mean ? 1.0 / fmax(n, 1.0) : 1.0;
    *loss = (float)(s * inv);
    stats[rows * kDistillStats] = (float)inv;
  }
}

template <class T>
__global__ __launch_bounds__(kT) void distill_bwd_k(DistillArgs a, int nseg, int seglen,
                                                    const float* __restrict__ dloss, int per_row, int past_caches,
                                                    typename T::store_t* __restrict__ dz) {
  constexpr int N = Piece<T>::kN;
  __shared__ int cls_s[kT];
  __shared__ float p_s[kT];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / nseg;
  const int begin = (int)(blockIdx.x % nseg) * seglen, end = min(a.V, begin + seglen);
  const auto* z = static_cast<const typename T::store_t*>(a.z) + row * a.ldz;
  const RowStats& st = reinterpret_cast<const RowStats*>(a.stats)[row];
  dz += row * a.V;
  if (st.used == 0.f) {  // a row that is left out: its logits are not looked at
    const Bytes16 zero = {{0, 0, 0, 0}};
    for (int i = begin + tid * N; i < end; i += kT * N) {
      if (i + N <= end) *reinterpret_cast<Bytes16*>(dz + i) = zero;
      else
        for (int e = i; e < end; ++e) dz[e] = 0;
    }
    return;
  }
  const float g = per_row ? dloss[row] : *dloss * a.stats[a.rows * kDistillStats];
  const double inv_t = 1.0 / a.temperature;
  const float c = (float)(kLog2e * inv_t), c1 = (float)kLog2e;
  const bool two = a.hard > 0 && a.temperature != 1.0;
  const float ref = st.ref, co = st.co, m = st.top, ci = st.ci, h1 = st.h1;
  // without a share (co = 0) a named class above `ref` must not make a NaN of an overflow
  const float lim = co == 0.f ? 0.f : INFINITY;
  constexpr int TILE = kT * kU * N;
  // a loop for each kind of access: of two stores under a condition the compiler makes one ordinary one
  auto sweep = [&](auto past) {
#pragma unroll 1
    for (int base = begin; base < end; base += TILE) {
      Piece<T> x[kU];
      load_tile<T, kT, past.value>(x, z, base, end);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int i = base + (u * kT + tid) * N;
        typename T::store_t o[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v = x[u].get(e);
          float d = co * fminf(exp2_raw((v - ref) * c), lim);
          if (two) d += h1 * exp2_raw((v - m) * c1);
          o[e] = T::store(g * d);
        }
        if (i + N <= end) {
          any16 w;
          __builtin_memcpy(&w, o, 16);
          if constexpr (past.value) __builtin_nontemporal_store(w, reinterpret_cast<any16*>(dz + i));
          else *reinterpret_cast<any16*>(dz + i) = w;
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (i + e < end) dz[i + e] = o[e];
        }
      }
    }
  };
  if (past_caches) sweep(std::true_type{});
  else sweep(std::false_type{});
  int cls;
  float t, v = 0.f, q = 0.f;
  load_entry(a, row, &cls, &t);
  cls_s[tid] = cls;
  double less = 0;  // p - q of an entry
  if (cls >= 0 && ci != 0.f) {
    v = T::load(z[cls]);
    q = ci * exp2f((v - m) * c);
    const double dt = (double)t - st.tref, d = (dt - ((double)v - m)) * inv_t + st.K;
    less = fabs(d) < 0.25 ? q * ((d - gain_near(d)) / (1.0 - d))
                          : (1 - a.hard) * a.temperature * exp(dt * inv_t - st.norm) - q;
  }
  p_s[tid] = (float)less;
  const int64_t y = a.hard > 0 ? load_int(a.target, row, a.target64) : -1;
  __syncthreads();  // also orders the stores above before the ones below
  if (cls >= begin && cls < end) {
    float more = 0, times = 0;  // a class that is named twice has both entries' share
    for (int j = 0; j < a.k; j += 8) {  // threads without an entry hold -1
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        more += cls_s[j + e] == cls ? p_s[j + e] : 0.f;
        times += cls_s[j + e] == cls ? 1.f : 0.f;
      }
    }
    float d = q * (1.f - times) - more;
    if (ci == 0.f) v = T::load(z[cls]);
    if (a.hard > 0) d += h1 * exp2f((v - m) * c1) - (cls == y ? (float)a.hard : 0.f);
    dz[cls] = T::store(g * d);
  }
  if (tid == 0 && y >= begin && y < end) {
    bool named = false;
    for (int j = 0; j < a.k; j += 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) named = named || cls_s[j + e] == y;
    }
    if (!named) {
      const float v = T::load(z[y]);
      float d = co * fminf(exp2f((v - ref) * c), lim);
      if (two) d += h1 * exp2f((v - m) * c1);
      dz[y] = T::store(g * (d - (float)a.hard));
    }
  }
}

void check_distill(const DistillArgs& a) {
  MX_CHECK(a.rows >= 0 && a.rows <= kMaxRows && a.V >= 1 && a.V <= (1 << 30) && a.k >= 1 && a.k <= kTopMax,
           "distill_loss: bad sizes");
  MX_CHECK(a.temperature > 0 && a.hard >= 0 && a.hard <= 1 && (a.hard == 0 || a.target), "distill_loss: bad weights");
}

}  // namespace

int64_t top_logits_scratch(int64_t rows, int V, int k) {
  const int nseg = row_segments(rows, V);
  return nseg > 1 ? rows * nseg * (k + 1) : 0;
}

void top_logits(const void* z, int type, int64_t ldz, int64_t rows, int V, int k, double temperature, void* values,
                int32_t* index, float* lse, void* scratch, hipStream_t st) {
  MX_CHECK(rows >= 0 && rows <= kMaxRows && V >= 1 && V <= (1 << 30) && k >= 1 && k <= kTopMax && k <= V &&
               temperature > 0,
           "top_logits: bad sizes");
  if (rows == 0) return;
  TopArgs a{z, values, index, lse, static_cast<uint64_t*>(scratch), ldz, rows, V, k, row_segments(rows, V), V,
            (float)(kLog2e / temperature), (float)(1.0 / temperature)};
  a.seglen = segment_length(V, &a.nseg);
  MX_CHECK(a.nseg == 1 || scratch, "top_logits: long rows need scratch");
  // one tile where a block's part of the row fits: a wave alone needs no barrier
  MX_BY_TYPE(type, T, {
    constexpr int wave_tile = 64 * kU * Piece<T>::kN;
    if (a.seglen <= wave_tile) launch_top<T, 64>(a, st);
    else launch_top<T, 256>(a, st);
    if (a.nseg > 1) MX_LAUNCH(top_merge_k<T>, dim3((uint32_t)rows), dim3(kT), 0, st, a);
  });
}

int64_t distill_scratch(int64_t rows, int V) {
  const int nseg = row_segments(rows, V);
  return nseg > 1 ? 8 * rows * nseg : 0;
}

void distill_fwd(const DistillArgs& a, float* loss_rows, float* loss, bool mean, void* scratch, hipStream_t st) {
  check_distill(a);
  int nseg = row_segments(a.rows, a.V);
  const int seglen = segment_length(a.V, &nseg);
  MX_CHECK(nseg == 1 || (scratch && (uintptr_t)scratch % 8 == 0), "distill_loss: long rows need scratch");
  auto launch = [&](auto type, auto far) {
    using T = decltype(type);
    constexpr bool FAR = far.value;
    double* part = nseg > 1 ? static_cast<double*>(scratch) : nullptr;
    MX_LAUNCH((distill_fwd_k<T, FAR>), dim3((uint32_t)(a.rows * nseg)), dim3(kT), 0, st, a, nseg, seglen, part, loss_rows);
    if (nseg > 1) MX_LAUNCH((distill_join_k<T, FAR>), dim3((uint32_t)a.rows), dim3(kT), 0, st, a, nseg, part, loss_rows);
  };
  if (a.rows > 0)
    MX_BY_TYPE(a.type, T, {
      if (a.temperature > kNearT) launch(T{}, std::true_type{});
      else launch(T{}, std::false_type{});
    });
  if (loss) MX_LAUNCH(distill_mean_k, dim3(1), dim3(1024), 0, st, loss_rows, a.stats, a.rows, mean ? 1 : 0, loss);
}

void distill_bwd(const DistillArgs& a, const float* dloss, bool per_row, void* dz, hipStream_t st) {
  check_distill(a);
  int nseg = row_segments(a.rows, a.V);
  const int seglen = segment_length(a.V, &nseg);
  // Past the caches, reads and writes: rows of whole cache lines that the last-level cache of 256 MB does
  // not hold.  A step (both directions) of 4096 x 131072 in bf16: 599 us, 615 with the writes alone, 667
  // with ordinary writes.  Other rows the other way round: 1023 x 50001 in fp16 40 us through the caches
  // and 46 past them, 4096 x 131071 in bf16 489 and 516 (partial lines are joined in the cache).
  const int64_t row_bytes = (int64_t)a.V * (a.type == kF32 ? 4 : 2);
  const bool past = ((uintptr_t)dz | (uintptr_t)row_bytes) % 128 == 0 && a.rows * row_bytes >= (256ll << 20);
  if (a.rows > 0)
    MX_BY_TYPE(a.type, T, MX_LAUNCH(distill_bwd_k<T>, dim3((uint32_t)(a.rows * nseg)), dim3(kT), 0, st, a, nseg,
                                    seglen, dloss, per_row ? 1 : 0, past ? 1 : 0,
                                    static_cast<typename T::store_t*>(dz)));
}

}  // namespace mx
