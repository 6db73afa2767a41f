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
  const bool odd = ((int)q & 1) != 0;
  if (r > h || (r == h && odd)) q += 1.f;
  else if (r < -h || (r == -h && odd)) q -= 1.f;
  return (int)q;
}

constexpr int kQT = 256;

template <class T>
__global__ __launch_bounds__(kQT) void quantize_rows_k(const typename T::store_t* __restrict__ x, int64_t ldx,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                                                       int K) {
  __shared__ uint32_t red[kQT / 64];
  const int64_t row = blockIdx.x;
  x += row * ldx;
  q += row * ldq;
  // the largest magnitude as bits: infinities and NaN are above every number
  uint32_t top = 0;
  for (int k = threadIdx.x; k < K; k += kQT) top = max(top, __float_as_uint(T::load(x[k])) & 0x7fffffffu);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQT / 64; ++w) top = max(top, red[w]);
  const bool ok = top < 0x7f800000u;
  const float s = ok ? fmaxf(__uint_as_float(top) / 127.f, kTiny) : __builtin_nanf("");
  const float inv = 1.f / s;
  for (int k = threadIdx.x; k < ldq; k += kQT) q[k] = ok && k < K ? (int8_t)quant1(T::load(x[k]), s, inv) : 0;
  if (threadIdx.x == 0) scale[row] = s;
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
  int N, K, relu, tiles_n;
};

// 64 channels x 64 tokens per block of four waves, 64 k per step
template <class T>
__global__ __launch_bounds__(256) void int8_gemm_k(GemmArgs a) {
  __shared__ __attribute__((aligned(16))) char sm[2][64 * 80];  // rows of 64 B at a pitch of 80
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = (blockIdx.x % a.tiles_n) * 64;
  const int64_t m0 = (int64_t)(blockIdx.x / a.tiles_n) * 64;
  const int lr = tid >> 2, lc = 16 * (tid & 3);
  const int8_t* wp = a.w + (int64_t)(n0 + lr) * a.ldw;
  const int8_t* qp = a.q + (m0 + lr) * a.ldq;
  const bool wok = n0 + lr < a.N, qok = m0 + lr < a.M;
  const int wn = (wave & 1) * 32, wm = (wave >> 1) * 32;
  i32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    const i32x4 vw = row16(wp, wok, k0 + lc, a.K), vq = row16(qp, qok, k0 + lc, a.K);
    __syncthreads();
    *reinterpret_cast<i32x4*>(sm[0] + lr * 80 + lc) = vw;
    *reinterpret_cast<i32x4*>(sm[1] + lr * 80 + lc) = vq;
    __syncthreads();
    i32x4 fw[2], fq[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 16 * i + (lane & 15), c = 16 * (lane >> 4);
      fw[i] = *reinterpret_cast<const i32x4*>(sm[0] + (wn + r) * 80 + c);
      fq[i] = *reinterpret_cast<const i32x4*>(sm[1] + (wm + r) * 80 + c);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fq[j], acc[i][j], 0, 0, 0);
  }
  typename T::store_t* y = static_cast<typename T::store_t*>(a.y);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t m = m0 + wm + 16 * j + (lane & 15);
    if (m >= a.M) continue;
    const float xs = a.xs[m];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + wn + 16 * i + 4 * (lane >> 4) + e;
        if (n >= a.N) continue;
        float v = (float)acc[i][j][e] * xs * a.ws[n];
        if (a.bias) v += a.bias[n];
        if (a.relu) v = v < 0.f ? 0.f : v;  // a NaN stays one
        y[m * a.N + n] = T::store(v);
      }
  }
}

}  // namespace

void quantize_rows(const void* x, int xtype, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int K,
                   hipStream_t st) {
  MX_CHECK(rows >= 0 && rows < (1ll << 31) && K >= 1 && ldq >= K, "quantize_rows: bad sizes");
  if (rows == 0) return;
  MX_BY_TYPE(xtype, T, MX_LAUNCH(quantize_rows_k<T>, dim3((uint32_t)rows), dim3(kQT), 0, st,
                                 static_cast<const typename T::store_t*>(x), ldx, q, ldq, scale, K));
}

void linear_int8(const int8_t* q, int64_t ldq, const float* xs, const int8_t* w, int64_t ldw, const float* ws,
                 const float* bias, void* y, int ytype, int64_t M, int N, int K, bool relu, hipStream_t st) {
  MX_CHECK(M >= 0 && N >= 1 && K >= 1 && K <= kInt8MaxK, "linear_int8: bad sizes");
  if (M == 0) return;
  GemmArgs a{q, w, xs, ws, bias, y, ldq, ldw, M, N, K, relu ? 1 : 0, cdiv(N, 64)};
  const int64_t blocks = (M + 63) / 64 * a.tiles_n;
  MX_CHECK(blocks < (1ll << 31), "linear_int8: too many tiles");
  MX_BY_TYPE(ytype, T, MX_LAUNCH(int8_gemm_k<T>, dim3((uint32_t)blocks), dim3(256), 0, st, a));
}

}  // namespace mx
