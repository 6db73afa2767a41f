// Linear layers in 8-bit integers: y = (q w^T) s_token s_channel + b, q = round(x / s_token).
//
// quantize_rows_k: one scale per row, s = max(max|x| / 127, 2^-126), q = x / s rounded half to even.
// The quotient is rounded as the exact one: rint(x * (1 / s)) is at most one step off, and the
// remainder x - q s, exact in fp32 by fma (x and q s are within one s of each other and multiples of
// the smaller one's last place), says which way.  Its double is compared with s: half of a small s
// need not be a number of fp32.
// int8_gemm_k: rows of q and rows of w, both contiguous in k, on v_mfma_i32_16x16x64_i8; the sum is a
// whole number below 2^31, so it is exact in any order.
#include <algorithm>
#include <type_traits>

#include "lowp.h"
#include "ops.h"

namespace mx {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kTiny = 1.17549435e-38f;  // 2^-126: its reciprocal is finite

__device__ __forceinline__ int quant1(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = __builtin_fmaf(-q, s, x), r2 = r + r;
  if (__builtin_expect(fabsf(r2) >= s, 0)) {
    const bool odd = ((int)q & 1) != 0;
    if (r2 > s || (r2 == s && odd)) q += 1.f;
    else if (r2 < -s || (r2 == -s && odd)) q -= 1.f;
  }
  return (int)q;
}

// A row's scale from its largest magnitude's bits.  Infinities and NaN are above every number.
struct RowScale {
  float s, inv;
  bool ok;
  __device__ __forceinline__ explicit RowScale(uint32_t top) {
    ok = top < 0x7f800000u;
    s = ok ? fmaxf(__uint_as_float(top) / 127.f, kTiny) : __builtin_nanf("");
    inv = 1.f / s;
  }
};
__device__ __forceinline__ uint32_t wave_max(uint32_t top) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  return top;
}

template <class T>
__device__ __forceinline__ void quant_piece(const Piece<T>& p, const RowScale& sc, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < Piece<T>::kN / 4; ++i) {
    w[i] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[i] |= (uint32_t)((sc.ok ? quant1(p.get(4 * i + e), sc.s, sc.inv) : 0) & 0xff) << (8 * e);
  }
}

// One row a block of TB threads.  Bound by its bytes: up to kQP pieces of 16 bytes a thread stay in
// registers between the maximum and the rounding; a longer row is read again, from the cache.  8192 x
// 8192 in bf16: 40 to 45 us, 4.5 to 5 TB/s.
constexpr int kQP = 4;

template <class T, int TB>
__global__ __launch_bounds__(TB) void quantize_rows_k(const typename T::store_t* __restrict__ x, int64_t ldx,
                                                      int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                                                      int K) {
  constexpr int N = Piece<T>::kN, TILE = TB * kQP * N;
  __shared__ uint32_t red[TB / 64];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  x += row * ldx;
  q += row * ldq;
  Piece<T> p[kQP];
  uint32_t top = 0;
  for (int k0 = 0; k0 < K; k0 += TILE) {
#pragma unroll
    for (int u = 0; u < kQP; ++u) p[u].load(x, k0 + (u * TB + tid) * N, K, 0);
#pragma unroll
    for (int u = 0; u < kQP; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(p[u].get(e)) & 0x7fffffffu);
  }
  top = wave_max(top);
  if constexpr (TB > 64) {
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TB / 64; ++w) top = max(top, red[w]);
  }
  const RowScale sc(top);
  if (tid == 0) scale[row] = sc.s;
  for (int k0 = 0; k0 < K; k0 += TILE) {
#pragma unroll
    for (int u = 0; u < kQP; ++u) {
      const int k = k0 + (u * TB + tid) * N;
      if (K > TILE) p[u].load(x, k, K, 0);
      uint32_t w[N / 4];
      quant_piece<T>(p[u], sc, w);
      if (k + N <= K) {
        __builtin_memcpy(q + k, w, N);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (k + e < K) q[k + e] = (int8_t)(w[e / 4] >> (8 * (e & 3)));
      }
    }
  }
  for (int k = K + tid; k < ldq; k += TB) q[k] = 0;
}

// 16 bytes of a row at k, zeros behind its end and for rows that do not exist
__device__ __forceinline__ i32x4 row16(const int8_t* p, bool row_ok, int k, int K) {
  i32x4 v = {0, 0, 0, 0};
  if (row_ok && k + 16 <= K) {
    const Bytes16 b = *reinterpret_cast<const Bytes16*>(p + k);
    v = i32x4{(int)b.v[0], (int)b.v[1], (int)b.v[2], (int)b.v[3]};
  } else if (row_ok && k < K) {
    uint32_t t[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) t[i >> 2] |= (uint32_t)(uint8_t)p[k + i] << (8 * (i & 3));
    v = i32x4{(int)t[0], (int)t[1], (int)t[2], (int)t[3]};
  }
  return v;
}

// 16 bytes at any address
__device__ __forceinline__ i32x4 load16(const int8_t* p) {
  const Bytes16 b = *reinterpret_cast<const Bytes16*>(p);
  return i32x4{(int)b.v[0], (int)b.v[1], (int)b.v[2], (int)b.v[3]};
}

// The 16 bytes at an address: at a multiple of 4 as they are, else from the five words that hold them
// (a word with a byte of a tensor lies in its allocation).  24 tokens of 8192 x 8191: 32 us, 60 with one
// read of 16 bytes at an odd address.
template <bool ODD>
struct Raw16 {
  i32x4 v;
  int more;
  __device__ __forceinline__ void load(const int8_t* p) {
    if constexpr (!ODD) {
      v = load16(p);
    } else {
      const uint32_t odd = (uint32_t)(uintptr_t)p & 3;
      const int8_t* q = p - odd;
      v = load16(q);
      more = *reinterpret_cast<const int*>(q + (odd ? 16 : 12));
    }
  }
  __device__ __forceinline__ i32x4 get(const int8_t* p) const {  // p: where it was loaded
    if constexpr (!ODD) return v;
    const uint32_t odd = (uint32_t)(uintptr_t)p & 3;
    return i32x4{(int)__builtin_amdgcn_alignbyte(v[1], v[0], odd), (int)__builtin_amdgcn_alignbyte(v[2], v[1], odd),
                 (int)__builtin_amdgcn_alignbyte(v[3], v[2], odd), (int)__builtin_amdgcn_alignbyte(more, v[3], odd)};
  }
};

// A piece that reaches `over` bytes behind the end of a row was read that much before its place, at
// the row's last 16 bytes: move it there, with zeros behind the end.
__device__ __forceinline__ i32x4 tail16(i32x4 v, int over) {
  if (over >= 16) return i32x4{0, 0, 0, 0};
  if (over <= 0) return v;
  if (over & 8) v = i32x4{v[2], v[3], 0, 0};
  if (over & 4) v = i32x4{v[1], v[2], v[3], 0};
  const uint32_t b = over & 3;
  return i32x4{(int)__builtin_amdgcn_alignbyte(v[1], v[0], b), (int)__builtin_amdgcn_alignbyte(v[2], v[1], b),
               (int)__builtin_amdgcn_alignbyte(v[3], v[2], b), (int)__builtin_amdgcn_alignbyte(0, v[3], b)};
}

struct GemmArgs {
  const int8_t* q;
  const int8_t* w;
  const float* xs;
  const float* ws;
  const float* bias;
  void* y;
  int64_t ldq, ldw, M;
  int N, K, relu, tiles_n, tiles_m;
};

// the epilogue of four channels of a token: their scales and biases, once for all tokens of a lane
struct Four {
  float ws[4], b[4];
  __device__ __forceinline__ Four(const GemmArgs& a, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = min(n + e, a.N - 1);
      ws[e] = a.ws[c];
      b[e] = a.bias ? a.bias[c] : 0.f;
    }
  }
  template <class T>
  __device__ __forceinline__ void put(const GemmArgs& a, int64_t m, int n, i32x4 acc, float xs) const {
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __builtin_fmaf((float)acc[e] * xs, ws[e], b[e]);
    // A token's scale with which the first product could leave fp32 at either end (|acc| < 2^31), though
    // the channel's scale brings it back: in 64 bits.
    if (__builtin_expect(!(fabsf(xs) >= kTiny && fabsf(xs) < 0x1p96f), 0)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = (float)((double)acc[e] * xs * ws[e] + b[e]);
    }
    typename T::store_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = T::store(a.relu && f[e] < 0.f ? 0.f : f[e]);  // a NaN stays one
    typename T::store_t* o = static_cast<typename T::store_t*>(a.y) + m * a.N + n;
    if (n + 3 < a.N) {
      __builtin_memcpy(o, v, sizeof(v));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) o[e] = v[e];
    }
  }
};

typedef __attribute__((address_space(3))) void lds_void_t;
// 16 bytes a lane straight to LDS (lane after lane from `lds`), from base + off.  A buffer instruction:
// the compiler takes a global one for an access through the flat path, which may touch LDS in any
// order, and would then wait for ALL of a wave's LDS reads before each use of one.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00027000);
}
__device__ __forceinline__ void glds16(__amdgpu_buffer_rsrc_t r, uint32_t off, int k0, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)lds, 16, (int)off, k0, 0, 0);
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// TM channels x TN tokens per block of WM x WN waves, 128 k a stage, NS stages in LDS.  A stage's rows
// are 128 bytes, a row's 16-byte pieces XOR-permuted by its number, so the fragments' reads (16 rows at
// one piece) spread over all banks.  DW, DQ: the channels' and the tokens' rows come straight from
// global memory (rows of whole, aligned pieces); else through registers (any alignment and K >= 16).
// Channels are the matrix instruction's rows: a lane ends with four of them for one token.
// The fragments of one half stage are read while the other half's are multiplied.  The barrier stands
// in the middle of a stage, where its second half is in registers: its buffer is free for stage
// t + NS there, and the first half of stage t + 1 is read behind it.  Reads, copies, loads and writes are
// issued one by one between the matrix instructions: a copy of 1 KB keeps its wave from issuing for 16
// cycles and more, and all of a stage's in a row leave the matrix units idle for half a stage (8192^3
// 447 us without it; 1777 x 5000 x 5000, whose rows go through registers, 84).
// Bound by the matrix units and their operands' way out of LDS: 8192^3 400 to 480 us by the card's clock,
// 2.3 to 2.75 POP/s, 60% of what the instruction alone reaches on such values; 1777 x 5000 x 5000 66 us,
// 1.35 POP/s (three quarters of the CUs have a tile).
template <class T, int TM, int TN, int WM, int WN, int NS, bool DW, bool DQ>
__global__ __launch_bounds__(64 * WM * WN) void int8_gemm_k(GemmArgs a) {
  constexpr int NW = WM * WN, FM = TM / WM / 16, FN = TN / WN / 16;
  constexpr int IA = TM / 8 / NW, IB = TN / 8 / NW;  // wave-wide copies of 1 KB a stage
  constexpr int SB = (TM + TN) * 128;
  static_assert((DW && DQ) || NS == 2, "through registers one stage is under way");
  __shared__ __attribute__((aligned(1024))) char sm[NS * SB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  // tiles in bands of kBand channel tiles, token by token: what runs together shares both operands
  constexpr int kBand = 8;
  const int band = bid / (kBand * a.tiles_m), in = bid % (kBand * a.tiles_m);
  const int bw = min(kBand, a.tiles_n - band * kBand);
  const int n0 = (band * kBand + in % bw) * TM;
  const int64_t m0 = (int64_t)(in / bw) * TN;
  const int8_t* wbase = a.w + (int64_t)n0 * a.ldw;
  const int8_t* qbase = a.q + m0 * a.ldq;
  const int chunk = 16 * ((lane & 7) ^ (lane >> 3));
  uint32_t offw[IA], offq[IB];
#pragma unroll
  for (int j = 0; j < IA; ++j)  // rows behind the last are the last: what they give is not stored
    offw[j] = (uint32_t)(min((wave * IA + j) * 8 + (lane >> 3), a.N - 1 - n0) * a.ldw) + chunk;
#pragma unroll
  for (int j = 0; j < IB; ++j)
    offq[j] = (uint32_t)(min<int64_t>((wave * IB + j) * 8 + (lane >> 3), a.M - 1 - m0) * a.ldq) + chunk;

  const auto rsw = tile_rsrc(wbase), rsq = tile_rsrc(qbase);
  i32x4 rw[DW ? 1 : IA], rq[DQ ? 1 : IB];
  // straight to LDS: copy j of a stage's
  constexpr int kCopies = (DW ? IA : 0) + (DQ ? IB : 0);
  auto copy = [&](int t, int buf, int j) {
    const int k0 = t * 128;
    // pieces behind the end of k are the stage's first: `clear` takes the tokens' side of them out
    const uint32_t back = k0 + chunk < a.K ? 0 : chunk;
    char* st = sm + buf * SB;
    const int i = DW ? j - IA : j;
    if (DW && j < IA) glds16(rsw, offw[j] - back, k0, st + (wave * IA + j) * 1024);
    else glds16(rsq, offq[i] - back, k0, st + TM * 128 + (wave * IB + i) * 1024);
  };
  auto fetch = [&](int t, int buf) {
#pragma unroll
    for (int j = 0; j < kCopies; ++j) copy(t, buf, j);
  };
  // to registers, and from there to LDS
  constexpr int kPieces = (DW ? 0 : IA) + (DQ ? 0 : IB);
  auto load = [&](int t, int j) {
    const int at = min(t * 128 + chunk, a.K - 16) - chunk;
    const int i = DW ? j : j - IA;
    if (!DW && j < IA) rw[j] = load16(wbase + at + offw[j]);
    else rq[i] = load16(qbase + at + offq[i]);
  };
  auto put = [&](auto end, int t, int buf, int j) {
    char* st = sm + buf * SB + lane * 16;
    const int i = DW ? j : j - IA;
    const bool w = !DW && j < IA;
    i32x4 v = w ? rw[j] : rq[i];
    if constexpr (end.value) v = tail16(v, max(t * 128 + chunk + 16 - a.K, 0));
    *reinterpret_cast<i32x4*>(st + (w ? (wave * IA + j) * 1024 : TM * 128 + (wave * IB + i) * 1024)) = v;
  };
  const int fr = lane & 15, fc = lane >> 4;
  const int rw0 = (wm * FM * 16 + fr) * 128, rq0 = TM * 128 + (wn * FN * 16 + fr) * 128;
  // fragment r of a half stage: the tokens' first
  auto read = [&](int buf, int half, int r, i32x4* fw, i32x4* fq) {
    const char* st = sm + buf * SB + 16 * ((4 * half + fc) ^ (fr & 7));
    if (r < FN) fq[r] = *reinterpret_cast<const i32x4*>(st + rq0 + r * 2048);
    else fw[r - FN] = *reinterpret_cast<const i32x4*>(st + rw0 + (r - FN) * 2048);
  };
  auto clear = [&](int t, int half, i32x4* fq) {
    if (DQ && t * 128 + 128 > a.K) {
      const bool ok = t * 128 + 64 * half + 16 * fc < a.K;
#pragma unroll
      for (int j = 0; j < FN; ++j) fq[j] = ok ? fq[j] : i32x4{0, 0, 0, 0};
    }
  };
  i32x4 acc[FM][FN] = {};
  // the products of (fw, fq); between them the reads of half a stage to (nw, nq) and `side`, a share at a time
  auto products = [&](auto more, const i32x4* fw, const i32x4* fq, int nbuf, int nhalf, i32x4* nw, i32x4* nq,
                      auto side) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if constexpr (more.value) {
#pragma unroll
        for (int r = i * (FM + FN) / FM; r < (i + 1) * (FM + FN) / FM; ++r) read(nbuf, nhalf, r, nw, nq);
      }
      side(i);
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fq[j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};

  const int nt = (a.K + 127) / 128;
  // through registers a stage is loaded in the second half of the last but one before it, and put in its
  // place in the first half of the one before it; the last stage is loaded again rather than under a
  // condition, which would make the compiler wait for it at once
  constexpr bool kDma = DW && DQ;
  constexpr int kAhead = kDma ? NS : 2;
  if constexpr (kDma) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
      if (s < nt) fetch(s, s);
    if (nt >= NS) wait_vm<(NS - 1) * (IA + IB)>();
    else wait_vm<0>();
  } else {
    fetch(0, 0);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) load(0, j);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) put(yes, 0, 0, j);
    wait_vm<0>();
    if (nt > 1) fetch(1, 1);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) load(min(1, nt - 1), j);
  }
  lds_barrier();
  i32x4 w0[FM], q0[FN], w1[FM], q1[FN];
#pragma unroll
  for (int r = 0; r < FM + FN; ++r) read(0, 0, r, w0, q0);
  int buf = 0;
  // a stage with another behind it, with or without one to copy (without: the other is the last)
  auto stage = [&](auto copies, int t) {
    const int next = buf + 1 == NS ? 0 : buf + 1;
    products(yes, w0, q0, buf, 1, w1, q1, [&](int i) {
#pragma unroll
      for (int j = i * kPieces / FM; j < (i + 1) * kPieces / FM; ++j) {
        if constexpr (copies.value) put(no, t + 1, next, j);
        else put(yes, t + 1, next, j);
      }
    });
    // stage t + 1 has landed; up to NS - 2 later ones are under way
    wait_vm<kDma && copies.value ? (NS - 2) * (IA + IB) : 0>();
    lds_barrier();
    products(yes, w1, q1, next, 0, w0, q0, [&](int i) {
      if constexpr (copies.value) {
#pragma unroll
        for (int j = i * kCopies / FM; j < (i + 1) * kCopies / FM; ++j) copy(t + kAhead, buf, j);
      }
#pragma unroll
      for (int j = i * kPieces / FM; j < (i + 1) * kPieces / FM; ++j) load(min(t + 2, nt - 1), j);
    });
    buf = next;
  };
  auto nothing = [](int) {};
  int t = 0;
  for (; t + kAhead < nt; ++t) stage(yes, t);
  for (; t + 1 < nt; ++t) stage(no, t);
  clear(t, 0, q0);
  products(yes, w0, q0, buf, 1, w1, q1, nothing);
  clear(t, 1, q1);
  products(no, w1, q1, 0, 0, w0, q0, nothing);
  float xs[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) xs[j] = a.xs[min<int64_t>(m0 + (wn * FN + j) * 16 + fr, a.M - 1)];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int n = n0 + (wm * FM + i) * 16 + 4 * fc;
    if (n >= a.N) continue;
    const Four four(a, n);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t m = m0 + (wn * FN + j) * 16 + fr;
      if (m < a.M) four.put<T>(a, m, n, acc[i][j], xs[j]);
    }
  }
}

template <class T, int TM, int TN, int WM, int WN, int NS>
void launch_gemm(GemmArgs a, bool dw, bool dq, hipStream_t st) {
  a.tiles_n = cdiv(a.N, TM);
  const int64_t tm = (a.M + TN - 1) / TN;
  MX_CHECK(tm * a.tiles_n <= kMaxRows, "linear_int8: too many tiles");
  a.tiles_m = (int)tm;
  const dim3 grid((uint32_t)(tm * a.tiles_n)), block(64 * WM * WN);
  if (dw && dq) MX_LAUNCH((int8_gemm_k<T, TM, TN, WM, WN, NS, true, true>), grid, block, 0, st, a);
  else if (dq) MX_LAUNCH((int8_gemm_k<T, TM, TN, WM, WN, 2, false, true>), grid, block, 0, st, a);
  else MX_LAUNCH((int8_gemm_k<T, TM, TN, WM, WN, 2, false, false>), grid, block, 0, st, a);
}

// Few tokens: bound by the weight's bytes.  A block of eight waves takes 16 FM channels and all of up
// to 16 FN tokens; each wave streams an eighth of k from global memory straight into the matrix
// instruction's operands (a lane has 16 bytes of one channel, 64 bytes of it lie in one instruction)
// and the sums, whole numbers, are added in LDS.  The tokens' rows are small and come from the caches.
// Left to itself the compiler waits for each product's operands soon after their loads.  ODD: rows of no
// alignment are read word by word.  With weights that no cache holds 1 x 8192 x 8192 takes 15 us (4.3
// TB/s), 24 tokens of it 20 us (3.3 TB/s: the blocks read as many bytes of the tokens as of the weight;
// 26 without the order of the loads, 23 with groups of four units, which take more than the nearest cache
// holds).
// QUANT: each block quantises the tokens for itself, to LDS: up to kQuantMax values cost it less than
// a launch before this one (one token of 4096 x 4096: 6.6 us with it, 10 without; 16 of 4096 x 1024: 7.5
// and 8.4), with the waves shared out among the tokens (21 us one token after the other).
constexpr int kSkinnyWaves = 8, kQuantMax = 16384;

template <class T, int FM, int FN, bool ODD, bool QUANT>
__global__ __launch_bounds__(64 * kSkinnyWaves) void int8_skinny_k(GemmArgs a, const typename T::store_t* x,
                                                                   int64_t ldx) {
  __shared__ i32x4 part[kSkinnyWaves][FM * FN][64];
  __shared__ __attribute__((aligned(16))) int8_t qs[QUANT ? kQuantMax + 16 * 80 : 16];
  __shared__ float xs_s[16];
  __shared__ uint32_t top_s[kSkinnyWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fc = lane >> 4;
  const int pitch = (a.K + 63) / 64 * 64 + 16;  // of a token's row in LDS
  if constexpr (QUANT) {
    constexpr int N = Piece<T>::kN;
    // waves of a token; 8 / per tokens at a time
    const int M = (int)a.M, per = M > 4 ? 1 : M > 2 ? 2 : M > 1 ? 4 : 8;
    const int first = wave / per * per, at = ((wave - first) * 64 + lane) * N;
    for (int m0 = 0; m0 < M; m0 += kSkinnyWaves / per) {
      const int m = m0 + wave / per, K = m < M ? a.K : 0;
      const typename T::store_t* xr = x + (int64_t)min(m, M - 1) * ldx;
      uint32_t top = 0;
      for (int k = at; k < K; k += per * 64 * N) {
        Piece<T> p;
        p.load(xr, k, K, 0);
#pragma unroll
        for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(p.get(e)) & 0x7fffffffu);
      }
      top = wave_max(top);
      if (lane == 0) top_s[wave] = top;
      __syncthreads();
      for (int w = 0; w < per; ++w) top = max(top, top_s[first + w]);
      const RowScale sc(top);
      if (m < M) {
        if (wave == first && lane == 0) xs_s[m] = sc.s;
        for (int k = at; k < pitch - 16; k += per * 64 * N) {
          Piece<T> p;
          p.load(xr, k, K, 0);  // zeros behind the end
          uint32_t w[N / 4];
          quant_piece<T>(p, sc, w);
          __builtin_memcpy(qs + m * pitch + k, w, N);
        }
      }
      __syncthreads();
    }
  }
  const int n0 = (blockIdx.x % a.tiles_n) * 16 * FM;
  const int64_t m0 = (int64_t)(blockIdx.x / a.tiles_n) * 16 * FN;
  const int8_t *pw[FM], *pq[FN];
  const int8_t* ql = qs + min(fr, QUANT ? (int)a.M - 1 : 0) * pitch + 16 * fc;
#pragma unroll
  for (int i = 0; i < FM; ++i) pw[i] = a.w + (int64_t)min(n0 + 16 * i + fr, a.N - 1) * a.ldw + 16 * fc;
#pragma unroll
  for (int j = 0; j < FN; ++j) pq[j] = a.q + min<int64_t>(m0 + 16 * j + fr, a.M - 1) * a.ldq + 16 * fc;
  i32x4 acc[FM][FN] = {};
  // a wave has groups of U units of 64 k, one after the other: with two a group takes a row's whole cache
  // lines, and one group is under way while the other is multiplied
  constexpr int U = 2;
  const int groups = ((a.K + 63) / 64 + U - 1) / U, each = (groups + kSkinnyWaves - 1) / kSkinnyWaves;
  struct Group {
    Raw16<ODD> w[U][FM], q[U][FN];
  };
  // a piece that reaches behind the end of k is read at the row's last 16 bytes
  auto at = [&](int g, int s) { return min(64 * (g * U + s) + 16 * fc, a.K - 16) - 16 * fc; };
  auto fetch = [&](Group& r, int g) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int s = 0; s < U; ++s) r.w[s][i].load(pw[i] + at(g, s));
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int s = 0; s < U; ++s) {
        if constexpr (QUANT) r.q[s][j].v = *reinterpret_cast<const i32x4*>(ql + min(64 * (g * U + s), pitch - 80));
        else r.q[s][j].load(pq[j] + at(g, s));
      }
    __builtin_amdgcn_sched_barrier(0);  // all of them under way before the group before it is waited for
  };
  auto use = [&](auto end, const Group& r, int g) {
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int over = max(64 * (g * U + s) + 16 * fc + 16 - a.K, 0);
      i32x4 fw[FM], fq[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        fw[i] = r.w[s][i].get(pw[i] + at(g, s));
        if constexpr (end.value) fw[i] = tail16(fw[i], over);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        fq[j] = QUANT ? r.q[s][j].v : r.q[s][j].get(pq[j] + at(g, s));
        if constexpr (end.value && !QUANT) fq[j] = tail16(fq[j], over);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fq[j], acc[i][j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  auto use_last = [&](const Group& r, int g) {
    if ((g + 1) * U * 64 <= a.K) use(no, r, g);
    else use(yes, r, g);
  };
  if (a.K >= 16) {
    int g = wave * each;
    const int last = min(groups, g + each);
    Group r0, r1;
    if (g < last) {
      fetch(r0, g);
      for (; g + 2 < last; g += 2) {
        fetch(r1, g + 1);
        use(no, r0, g);
        fetch(r0, g + 2);
        use(no, r1, g + 1);
      }
      if (g + 1 < last) {
        fetch(r1, g + 1);
        use(no, r0, g);
        use_last(r1, g + 1);
      } else {
        use_last(r0, g);
      }
    }
  } else if (wave == 0) {
    i32x4 fw[FM], fq[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) fw[i] = row16(pw[i] - 16 * fc, true, 16 * fc, a.K);
#pragma unroll
    for (int j = 0; j < FN; ++j)
      fq[j] = QUANT ? *reinterpret_cast<const i32x4*>(ql) : row16(pq[j] - 16 * fc, true, 16 * fc, a.K);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fq[j], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) part[wave][i * FN + j][lane] = acc[i][j];
  __syncthreads();
  for (int f = tid; f < FM * FN * 64; f += 64 * kSkinnyWaves) {
    const int g = f >> 6, l = f & 63, i = g / FN, j = g % FN;
    i32x4 v = part[0][g][l];
#pragma unroll
    for (int w = 1; w < kSkinnyWaves; ++w) v += part[w][g][l];
    const int64_t m = m0 + 16 * j + (l & 15);
    const int n = n0 + 16 * i + 4 * (l >> 4);
    if (m < a.M && n < a.N) Four(a, n).put<T>(a, m, n, v, QUANT ? xs_s[m] : a.xs[m]);
  }
}

template <class T, int FM, int FN, bool QUANT = false>
void launch_skinny(GemmArgs a, hipStream_t st, const void* x = nullptr, int64_t ldx = 0) {
  a.tiles_n = cdiv(a.N, 16 * FM);
  // as many tokens a launch as its grid takes
  const int64_t M = a.M, most = std::max<int64_t>(kMaxRows / a.tiles_n, 1) * 16 * FN;
  for (int64_t m = 0; m < M; m += most) {
    a.M = std::min(most, M - m);
    const int64_t blocks = (a.M + 16 * FN - 1) / (16 * FN) * a.tiles_n;
    MX_CHECK(blocks <= kMaxRows, "linear_int8: too many tiles");
    const dim3 grid((uint32_t)blocks), block(64 * kSkinnyWaves);
    const auto* xt = static_cast<const typename T::store_t*>(x);
    auto aligned = [&](const int8_t* p, int64_t ld) { return ((uintptr_t)p | (uintptr_t)ld | (uintptr_t)a.K) % 4 == 0; };
    const bool odd = !aligned(a.w, a.ldw) || (!QUANT && !aligned(a.q, a.ldq));
    if (odd) MX_LAUNCH((int8_skinny_k<T, FM, FN, true, QUANT>), grid, block, 0, st, a, xt, ldx);
    else MX_LAUNCH((int8_skinny_k<T, FM, FN, false, QUANT>), grid, block, 0, st, a, xt, ldx);
    if constexpr (!QUANT) {
      a.q += a.M * a.ldq;
      a.xs += a.M;
    }
    a.y = static_cast<typename T::store_t*>(a.y) + a.M * a.N;
  }
}

}  // namespace

void quantize_rows(const void* x, int xtype, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int K,
                   hipStream_t st) {
  MX_CHECK(rows >= 0 && rows <= kMaxRows && K >= 1 && K <= kMaxLength && ldq >= K, "quantize_rows: bad sizes");
  if (rows == 0) return;
  // one wave where a row fits its registers: no barrier
  MX_BY_TYPE(xtype, T, {
    using E = typename T::store_t;
    const dim3 grid((uint32_t)rows);
    if (K <= 64 * kQP * Piece<T>::kN)
      MX_LAUNCH((quantize_rows_k<T, 64>), grid, dim3(64), 0, st, static_cast<const E*>(x), ldx, q, ldq, scale, K);
    else
      MX_LAUNCH((quantize_rows_k<T, 256>), grid, dim3(256), 0, st, static_cast<const E*>(x), ldx, q, ldq, scale, K);
  });
}

void linear_int8(const int8_t* q, int64_t ldq, int q_room, const float* xs, const int8_t* w, int64_t ldw, int w_room,
                 const float* ws, const float* bias, void* y, int ytype, int64_t M, int N, int K, bool relu,
                 hipStream_t st) {
  MX_CHECK(M >= 0 && M <= kMaxRows && N >= 1 && N <= kMaxLength && K >= 1 && K <= kInt8MaxK,
           "linear_int8: bad sizes");
  MX_CHECK(ldq >= 0 && ldq <= kInt8MaxLd && ldw >= 0 && ldw <= kInt8MaxLd, "linear_int8: row stride too large");
  if (M == 0) return;
  GemmArgs a{q, w, xs, ws, bias, y, ldq, ldw, M, N, K, relu ? 1 : 0, 0, 0};
  auto whole = [K](const void* p, int64_t ld, int room) {
    return ((uintptr_t)p | (uintptr_t)ld) % 16 == 0 && room >= (K + 15) / 16 * 16;
  };
  const bool dw = whole(w, ldw, w_room), dq = whole(q, ldq, q_room);
  // A tile kernel's time is its rounds over the machine times the time of a stage, in us as measured at
  // K of 4096 to 8192 (copied straight to LDS; through registers, between rows of 16 bytes and odd ones):
  // 64 x 64 with two blocks a CU 0.55 (0.8), 128 x 128 with one and four stages in LDS 0.72, with two and
  // two stages 1.1 (1.45), 192 channels x 256 tokens 1.6 (1.8), 256 x 256 1.8 (2.35).  So 512 x 4096 x
  // 4096 takes 17 us on the smallest (25 on 128 x 128), 1777 x 5008 x 5008 60 us on 192 x 256 (69 on 256 x
  // 256, 87 on 128 x 128), and 4096^3 60 us on the largest (81 on 192 x 256); of odd rows 1024 x 4096 x
  // 4095 42 us on 128 x 128 (63 on 64 x 64 and on 192 x 256), 4096 x 4096 x 4095 83 us on the largest (122
  // on 128 x 128 and on 192 x 256).
  const int64_t cu = device_cu_count();
  auto rounds = [&](int tn, int tm, int64_t slots) {
    const int64_t tiles = (M + tm - 1) / tm * cdiv(N, tn);
    return (double)((tiles + slots - 1) / slots);
  };
  const bool dma = dw && dq;
  const double cost[5] = {(dma ? 0.55 : 0.8) * rounds(64, 64, 2 * cu), dma ? 0.72 * rounds(128, 128, cu) : 1e30,
                          (dma ? 1.1 : 1.45) * rounds(128, 128, 2 * cu), (dma ? 1.6 : 1.8) * rounds(192, 256, cu),
                          (dma ? 1.8 : 2.35) * rounds(256, 256, cu)};
  const int best = (int)(std::min_element(cost, cost + 5) - cost);
  MX_BY_TYPE(ytype, T, {
    // Few tokens: the weight's bytes, and for each block the tokens'.  Twice the channels a block halve
    // the latter, where that leaves a block a CU: 16 tokens of 8192 x 8192 19 us (21 without), of 4096 x
    // 4096 9.0 us (7.4 without); 32 tokens of 32000 x 4096 42 us (55 without), of 4096 x 4096 9 us, on
    // tiles 19.  Four times where that leaves one: 32 tokens of 16384 x 8192 34 us (38 with twice), of 32000
    // x 4095 49 us (58).  Up to 16 tokens it changes nothing.
    const bool wide = M > 8 && N >= 32 * cu;
    if (M <= 16 || K < 16) {
      if (wide) launch_skinny<T, 2, 1>(a, st);
      else launch_skinny<T, 1, 1>(a, st);
    } else if (M <= 32) {
      if (N >= 64 * cu) launch_skinny<T, 4, 2>(a, st);
      else if (wide) launch_skinny<T, 2, 2>(a, st);
      else launch_skinny<T, 1, 2>(a, st);
    } else if (best == 0) launch_gemm<T, 64, 64, 2, 2, 4>(a, dw, dq, st);
    else if (best == 1) launch_gemm<T, 128, 128, 2, 4, 4>(a, dw, dq, st);
    else if (best == 2) launch_gemm<T, 128, 128, 2, 4, 2>(a, dw, dq, st);
    else if (best == 3) launch_gemm<T, 192, 256, 2, 4, 2>(a, dw, dq, st);
    else launch_gemm<T, 256, 256, 2, 4, 2>(a, dw, dq, st);
  });
}

namespace {
// tokens that the product's own kernel quantises
bool quantises(int xtype, int ytype, int64_t M, int K) { return xtype == ytype && M <= 16 && M * K <= kQuantMax; }
int64_t padded(int K) { return (K + 15) / 16 * 16; }
}  // namespace

int64_t linear_int8_scratch(int xtype, int ytype, int64_t M, int K) {
  return quantises(xtype, ytype, M, K) ? 0 : M * (padded(K) + 4);
}

void linear_int8_float(const void* x, int xtype, int64_t ldx, const int8_t* w, int64_t ldw, int w_room, const float* ws,
                       const float* bias, void* y, int ytype, int64_t M, int N, int K, bool relu, void* scratch,
                       hipStream_t st) {
  MX_CHECK(M >= 0 && M <= kMaxRows && N >= 1 && N <= kMaxLength && K >= 1 && K <= kInt8MaxK && ldw >= 0 &&
               ldw <= kInt8MaxLd,
           "linear_int8: bad sizes");
  if (M == 0) return;
  if (quantises(xtype, ytype, M, K)) {
    GemmArgs a{nullptr, w, nullptr, ws, bias, y, 0, ldw, M, N, K, relu ? 1 : 0, 0, 0};
    MX_BY_TYPE(ytype, T, (launch_skinny<T, 1, 1, true>(a, st, x, ldx)));
    return;
  }
  MX_CHECK(scratch, "linear_int8: scratch needed");
  int8_t* q = static_cast<int8_t*>(scratch);
  float* s = reinterpret_cast<float*>(q + M * padded(K));
  quantize_rows(x, xtype, ldx, q, padded(K), s, M, K, st);
  linear_int8(q, padded(K), (int)padded(K), s, w, ldw, w_room, ws, bias, y, ytype, M, N, K, relu, st);
}

}  // namespace mx
