// Linear layers in 8-bit integers: y = (q w^T) s_token s_channel + b, q = round(x / s_token).
//
// quantize_rows_k: one scale per row, s = max(max|x| / 127, 2^-126), q = x / s rounded half to even.
// The quotient is rounded as the exact one: rint(x * (1 / s)) is at most one step off, and the
// remainder x - q s, exact in fp32 by fma (x and q s are within one s of each other and multiples of
// the smaller one's last place), says which way.
// int8_gemm_k: rows of q and rows of w, both contiguous in k, on v_mfma_i32_16x16x64_i8; the sum is a
// whole number below 2^31, so it is exact in any order.
#include "lowp.h"
#include "ops.h"

namespace mx {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kTiny = 1.17549435e-38f;  // 2^-126: its reciprocal is finite

__device__ __forceinline__ int quant1(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
  if (__builtin_expect(fabsf(r) >= h, 0)) {
    const bool odd = ((int)q & 1) != 0;
    if (r > h || (r == h && odd)) q += 1.f;
    else if (r < -h || (r == -h && odd)) q -= 1.f;
  }
  return (int)q;
}

// One row a block of TB threads.  Bound by its bytes: up to kQP pieces of 16 bytes a thread stay in
// registers between the maximum and the rounding; a longer row is read again, from the cache.
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
  // the largest magnitude as bits: infinities and NaN are above every number
  uint32_t top = 0;
  for (int k0 = 0; k0 < K; k0 += TILE) {
#pragma unroll
    for (int u = 0; u < kQP; ++u) p[u].load(x, k0 + (u * TB + tid) * N, K, 0);
#pragma unroll
    for (int u = 0; u < kQP; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(p[u].get(e)) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if constexpr (TB > 64) {
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TB / 64; ++w) top = max(top, red[w]);
  }
  const bool ok = top < 0x7f800000u;
  const float s = ok ? fmaxf(__uint_as_float(top) / 127.f, kTiny) : __builtin_nanf("");
  const float inv = 1.f / s;
  if (tid == 0) scale[row] = s;
  for (int k0 = 0; k0 < K; k0 += TILE) {
#pragma unroll
    for (int u = 0; u < kQP; ++u) {
      const int k = k0 + (u * TB + tid) * N;
      if (K > TILE) p[u].load(x, k, K, 0);
      uint32_t w[N / 4];
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        w[i] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[i] |= (uint32_t)((ok ? quant1(p[u].get(4 * i + e), s, inv) : 0) & 0xff) << (8 * e);
      }
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

__device__ uint4 g_zero16;
typedef __attribute__((address_space(3))) void lds_void_t;
__device__ __forceinline__ void glds16(const void* src, void* lds) {
  __builtin_amdgcn_global_load_lds(src, (lds_void_t*)lds, 16, 0, 0);
}

// TM channels x TN tokens per block of WM x WN waves, 128 k a stage, two stages in LDS.  A stage's
// rows are 128 bytes, a row's 16-byte pieces XOR-permuted by its number, so the fragments' reads (16
// rows at one piece) spread over all banks.  DMA: the stage comes straight from global memory
// (rows of whole, aligned pieces); else through registers (any alignment, the ragged end of k in
// bytes).  Channels are the matrix instruction's rows: a lane ends with four of them for one token.
template <class T, int TM, int TN, int WM, int WN, bool DMA>
__global__ __launch_bounds__(64 * WM * WN) void int8_gemm_k(GemmArgs a) {
  constexpr int NW = WM * WN, FM = TM / WM / 16, FN = TN / WN / 16;
  constexpr int IA = TM / 8 / NW, IB = TN / 8 / NW;  // wave-wide copies of 1 KB a stage
  constexpr int SB = (TM + TN) * 128;
  __shared__ __attribute__((aligned(1024))) char sm[2 * SB];
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

  i32x4 rw[DMA ? 1 : IA], rq[DMA ? 1 : IB];
  auto fetch = [&](int t) {
    const int k0 = t * 128;
    if constexpr (DMA) {
      char* st = sm + (t & 1) * SB;
      if (k0 + 128 <= a.K) {
#pragma unroll
        for (int j = 0; j < IA; ++j) glds16(wbase + k0 + offw[j], st + (wave * IA + j) * 1024);
#pragma unroll
        for (int j = 0; j < IB; ++j) glds16(qbase + k0 + offq[j], st + TM * 128 + (wave * IB + j) * 1024);
      } else {
        const bool ok = k0 + chunk < a.K;
        const void* zero = &g_zero16;
#pragma unroll
        for (int j = 0; j < IA; ++j) glds16(ok ? wbase + k0 + offw[j] : zero, st + (wave * IA + j) * 1024);
#pragma unroll
        for (int j = 0; j < IB; ++j) glds16(ok ? qbase + k0 + offq[j] : zero, st + TM * 128 + (wave * IB + j) * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < IA; ++j) rw[j] = row16(wbase + (offw[j] - chunk), true, k0 + chunk, a.K);
#pragma unroll
      for (int j = 0; j < IB; ++j) rq[j] = row16(qbase + (offq[j] - chunk), true, k0 + chunk, a.K);
    }
  };
  auto put = [&](int t) {
    if constexpr (!DMA) {
      char* st = sm + (t & 1) * SB + lane * 16;
#pragma unroll
      for (int j = 0; j < IA; ++j) *reinterpret_cast<i32x4*>(st + (wave * IA + j) * 1024) = rw[j];
#pragma unroll
      for (int j = 0; j < IB; ++j) *reinterpret_cast<i32x4*>(st + TM * 128 + (wave * IB + j) * 1024) = rq[j];
    }
  };

  i32x4 acc[FM][FN] = {};
  const int nt = (a.K + 127) / 128;
  fetch(0);
  put(0);
  const int fr = lane & 15, fc = lane >> 4;
  for (int t = 0; t < nt; ++t) {
    if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // stage t is there for every wave, and stage t - 1 is used up
    if (t + 1 < nt) fetch(t + 1);
    const char* sw = sm + (t & 1) * SB + (wm * FM * 16 + fr) * 128;
    const char* sq = sm + (t & 1) * SB + TM * 128 + (wn * FN * 16 + fr) * 128;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int c = 16 * ((4 * ks + fc) ^ (fr & 7));
      i32x4 fw[FM], fq[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fw[i] = *reinterpret_cast<const i32x4*>(sw + i * 2048 + c);
#pragma unroll
      for (int j = 0; j < FN; ++j) fq[j] = *reinterpret_cast<const i32x4*>(sq + j * 2048 + c);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fq[j], acc[i][j], 0, 0, 0);
    }
    if (t + 1 < nt) put(t + 1);
  }
  typename T::store_t* y = static_cast<typename T::store_t*>(a.y);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int n = n0 + (wm * FM + i) * 16 + 4 * fc;
    float ws[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ws[e] = n + e < a.N ? a.ws[n + e] : 0.f;
      b[e] = a.bias && n + e < a.N ? a.bias[n + e] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t m = m0 + (wn * FN + j) * 16 + fr;
      if (m >= a.M) continue;
      const float xs = a.xs[m];
      typename T::store_t v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f = (float)acc[i][j][e] * xs * ws[e] + b[e];
        v[e] = T::store(a.relu && f < 0.f ? 0.f : f);  // a NaN stays one
      }
      typename T::store_t* o = y + m * a.N + n;
      if (n + 3 < a.N) {
        __builtin_memcpy(o, v, sizeof(v));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.N) o[e] = v[e];
      }
    }
  }
}

template <class T, int TM, int TN, int WM, int WN>
void launch_gemm(GemmArgs a, bool dma, hipStream_t st) {
  a.tiles_n = cdiv(a.N, TM);
  const int64_t tm = (a.M + TN - 1) / TN;
  MX_CHECK(tm * a.tiles_n < (1ll << 31) / 8, "linear_int8: too many tiles");
  a.tiles_m = (int)tm;
  const dim3 grid((uint32_t)(tm * a.tiles_n)), block(64 * WM * WN);
  if (dma) MX_LAUNCH((int8_gemm_k<T, TM, TN, WM, WN, true>), grid, block, 0, st, a);
  else MX_LAUNCH((int8_gemm_k<T, TM, TN, WM, WN, false>), grid, block, 0, st, a);
}

}  // namespace

void quantize_rows(const void* x, int xtype, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int K,
                   hipStream_t st) {
  MX_CHECK(rows >= 0 && rows < (1ll << 31) && K >= 1 && ldq >= K, "quantize_rows: bad sizes");
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

void linear_int8(const int8_t* q, int64_t ldq, const float* xs, const int8_t* w, int64_t ldw, const float* ws,
                 const float* bias, void* y, int ytype, int64_t M, int N, int K, bool relu, hipStream_t st) {
  MX_CHECK(M >= 0 && N >= 1 && K >= 1 && K <= kInt8MaxK, "linear_int8: bad sizes");
  MX_CHECK(ldq >= 0 && ldq <= kInt8MaxLd && ldw >= 0 && ldw <= kInt8MaxLd, "linear_int8: row stride too large");
  if (M == 0) return;
  GemmArgs a{q, w, xs, ws, bias, y, ldq, ldw, M, N, K, relu ? 1 : 0, 0, 0};
  auto whole = [](const void* p, int64_t ld) { return ((uintptr_t)p | (uintptr_t)ld) % 16 == 0; };
  const bool dma = K % 16 == 0 && whole(q, ldq) && whole(w, ldw);
  MX_BY_TYPE(ytype, T, {
    if (M >= 1024 && N >= 1024) launch_gemm<T, 256, 256, 2, 4>(a, dma, st);
    else launch_gemm<T, 128, 128, 2, 2>(a, dma, st);
  });
}

}  // namespace mx
