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

// running (maximum, sum of exp2((z - m) c))
struct MaxSum {
  float m = kLowest, s = 0.f;
  __device__ __forceinline__ void add(float z, float c) {
    if (z > m) {
      s *= exp2f((m - z) * c);
      m = z;
    }
    s += exp2f((z - m) * c);
  }
  __device__ __forceinline__ void merge(float om, float os, float c) {
    const float n = fmaxf(m, om);
    s = s * exp2f((m - n) * c) + os * exp2f((om - n) * c);
    m = n;
  }
};

constexpr int kT = 256;

// over a block of kT threads; every thread gets the result
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
  for (int w = 0; w < kT / 64; ++w) t.merge(red[2 * w], red[2 * w + 1], c);
  return t;
}

template <class T>
__global__ __launch_bounds__(kT) void top_logits_k(const typename T::store_t* __restrict__ z, int64_t ldz, int V,
                                                   int k, float c, float inv_t, typename T::store_t* __restrict__ val,
                                                   int32_t* __restrict__ idx, float* __restrict__ lse) {
  __shared__ float red[2 * kT / 64];
  __shared__ uint64_t rk[kT / 64];
  const int64_t row = blockIdx.x;
  z += row * ldz;
  MaxSum ms;
  for (int i = threadIdx.x; i < V; i += kT) ms.add(T::load(z[i]), c);
  ms = block_merge(ms, c, red);
  uint64_t last = ~0ull;
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < V; i += kT) {
      const uint64_t key = order_key(T::load(z[i]), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, o, 64);
      best = other > best ? other : best;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) rk[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kT / 64; ++w) best = rk[w] > best ? rk[w] : best;
    last = best;
    if (threadIdx.x == 0) {
      const uint32_t i = key_index(best);
      val[row * k + j] = z[i];
      idx[row * k + j] = (int32_t)i;
      if (j == 0) {
        const float v = T::load(z[i]);
        // an infinite or NaN maximum is the sum's value; of a row of -inf as well
        const bool fin = v - v == 0.f;
        lse[row] = fin ? ms.m * inv_t + logf(ms.s) : v;
      }
    }
  }
}

__device__ __forceinline__ int64_t load_int(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ double block_sum_d(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0;
  for (int w = 0; w < kT / 64; ++w) t += red[w];
  return t;
}

// what a row's named entries are: class (or -1) and t_j / T; k <= kT, one entry a thread
__device__ __forceinline__ void load_entry(const DistillArgs& a, int64_t row, double inv_t, int* cls, double* u) {
  *cls = -1;
  *u = 0;
  if ((int)threadIdx.x >= a.k) return;
  const int64_t c = load_int(a.ti, row * a.k + threadIdx.x, a.ti64);
  const float t = load_any(a.tv, row * a.k + threadIdx.x, a.tv_type);
  if (c >= 0 && c < a.V && !(t == -INFINITY)) {
    *cls = (int)c;
    *u = (double)t * inv_t;
  }
}

constexpr int kMaskBits = 1 << 17;  // named classes are marked in LDS, this many classes at a time

template <class T>
__global__ __launch_bounds__(kT) void distill_fwd_k(DistillArgs a, float* __restrict__ loss_rows) {
  __shared__ float red[2 * kT / 64];
  __shared__ double redd[kT / 64];
  __shared__ int cls_s[kT];
  __shared__ uint32_t mask[kMaskBits / 32];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const auto* z = static_cast<const typename T::store_t*>(a.z) + row * a.ldz;
  float* st = a.stats + row * kDistillStats;
  const double inv_t = 1.0 / a.temperature;
  const float c = (float)(kLog2e * inv_t), c1 = (float)kLog2e;
  int cls;
  double u;
  load_entry(a, row, inv_t, &cls, &u);
  cls_s[tid] = cls;
  const bool any = __syncthreads_or(cls >= 0);
  const int64_t y = a.target ? load_int(a.target, row, a.target64) : -1;
  const bool counted = a.target ? y >= 0 && y < a.V : any;
  if (!counted) {
    if (tid == 0) loss_rows[row] = 0.f;
    if (tid < kDistillStats) st[tid] = 0.f;
    return;
  }
  bool first = cls >= 0;  // not named by an earlier entry
  for (int j = 0; j < a.k && j < tid; ++j) first = first && cls_s[j] != cls;
  // the classes outside (with the teacher's lse) or all of them
  const bool tail = a.tlse != nullptr;
  const bool two = a.hard > 0 && a.temperature != 1.0;
  MaxSum out, one;
  for (int v0 = 0; v0 < a.V; v0 += kMaskBits) {
    const int n = min(a.V - v0, kMaskBits);
    if (tail) {
      __syncthreads();
      for (int i = tid; i < (n + 31) / 32; i += kT) mask[i] = 0;
      __syncthreads();
      if (cls >= v0 && cls < v0 + n) atomicOr(&mask[(cls - v0) >> 5], 1u << ((cls - v0) & 31));
      __syncthreads();
    }
    for (int i = tid; i < n; i += kT) {
      const float v = T::load(z[v0 + i]);
      if (!tail || !((mask[i >> 5] >> (i & 31)) & 1)) out.add(v, c);
      if (two) one.add(v, c1);
    }
  }
  out = block_merge(out, c, red);
  if (two) one = block_merge(one, c1, red);
  // all classes: those outside and the named ones, each once
  MaxSum in;
  const float zc = cls >= 0 ? T::load(z[cls]) : 0.f;
  if (tail && first) in.add(zc, c);
  in = block_merge(in, c, red);
  MaxSum all = out;
  if (tail) all.merge(in.m, in.s, c);
  if (two) { one.s *= exp2f((one.m - all.m) * c1); one.m = all.m; }
  const double log_z = log((double)all.s);
  // the teacher
  double norm = 0;
  if (tail) norm = a.tlse[row];
  else if (any) {
    double most = cls >= 0 ? u : -INFINITY;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmax(most, __shfl_xor(most, o, 64));
    __syncthreads();
    if ((tid & 63) == 0) redd[tid >> 6] = most;
    __syncthreads();
    for (int w = 0; w < kT / 64; ++w) most = fmax(most, redd[w]);
    norm = most + log(block_sum_d(cls >= 0 ? exp(u - most) : 0.0, redd));
  }
  const double p = cls >= 0 ? exp(u - norm) : 0.0;
  // p = 0 has no term, whatever the student's value
  double kd = block_sum_d(p == 0 ? 0.0 : p * ((u - norm) - (((double)zc - all.m) * inv_t - log_z)), redd);
  const double named = block_sum_d(p, redd);
  if (tid != 0) return;
  // exp2((z - out.m) c) * co: the share of a class outside
  const bool has_out = out.s > 0.f || out.s != out.s;
  double mass = tail ? named : any ? 1.0 : 0.0, rest = 0.0;
  const double shift = ((double)out.m - all.m) * inv_t;
  if (tail && has_out && !(named >= 1)) {
    rest = 1.0 - named;
    kd += rest * (log(rest) - (shift + log((double)out.s) - log_z));
    mass = 1.0;
  }
  const double co = has_out ? mass * exp(shift) / all.s - (tail ? rest / out.s : 0.0)
                    : all.s > 0.f ? 0.0 : __builtin_nan("");  // a row of -inf has no distribution
  const float ref = has_out ? out.m : all.m;
  const double h = a.hard, z1 = two ? (double)one.s : (double)all.s;
  double loss = (1 - h) * a.temperature * a.temperature * kd;
  if (h > 0) loss += h * (log(z1) - ((double)T::load(z[y]) - all.m));
  loss_rows[row] = (float)loss;
  const double w = (1 - h) * a.temperature;
  st[0] = ref;
  st[1] = (float)(w * co + (h > 0 && !two ? h * exp((double)ref - all.m) / z1 : 0.0));
  st[2] = all.m;
  st[3] = any ? (float)(w * mass / all.s) : 0.f;
  st[4] = h > 0 ? (float)(h / z1) : 0.f;
  st[5] = 1.f;
  const float hi = (float)norm;
  st[6] = hi;
  st[7] = (float)(norm - hi);
}

// loss = the sum or mean of the rows' losses; the rows' weight goes behind their statistics
__global__ __launch_bounds__(kT) void distill_mean_k(const float* __restrict__ loss_rows, float* __restrict__ stats,
                                                     int64_t rows, int mean, float* __restrict__ loss) {
  __shared__ double red[kT / 64];
  double s = 0, n = 0;
  for (int64_t i = threadIdx.x; i < rows; i += kT) {
    s += loss_rows[i];
    n += stats[i * kDistillStats + 5];
  }
  s = block_sum_d(s, red);
  n = block_sum_d(n, red);
  if (threadIdx.x == 0) {
    const double inv = mean ? 1.0 / fmax(n, 1.0) : 1.0;
    *loss = (float)(s * inv);
    stats[rows * kDistillStats] = (float)inv;
  }
}

template <class T>
__global__ __launch_bounds__(kT) void distill_bwd_k(DistillArgs a, const float* __restrict__ dloss, int per_row,
                                                    typename T::store_t* __restrict__ dz) {
  __shared__ int cls_s[kT];
  __shared__ float p_s[kT];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const auto* z = static_cast<const typename T::store_t*>(a.z) + row * a.ldz;
  const float* st = a.stats + row * kDistillStats;
  dz += row * a.V;
  if (st[5] == 0.f) {
    for (int i = tid; i < a.V; i += kT) dz[i] = T::store(0.f);
    return;
  }
  const float g = per_row ? dloss[row] : *dloss * a.stats[a.rows * kDistillStats];
  const double inv_t = 1.0 / a.temperature;
  const float c = (float)(kLog2e * inv_t), c1 = (float)kLog2e;
  const bool two = a.hard > 0 && a.temperature != 1.0;
  const float ref = st[0], co = st[1], m = st[2], ci = st[3], h1 = st[4];
  for (int i = tid; i < a.V; i += kT) {
    const float v = T::load(z[i]);
    float d = co == 0.f ? 0.f : co * exp2f((v - ref) * c);
    if (two) d += h1 * exp2f((v - m) * c1);
    dz[i] = T::store(g * d);
  }
  int cls;
  double u;
  load_entry(a, row, inv_t, &cls, &u);
  cls_s[tid] = cls;
  p_s[tid] = cls >= 0 ? (float)((1 - a.hard) * a.temperature * exp(u - st[6] - st[7])) : 0.f;
  const int64_t y = a.hard > 0 ? load_int(a.target, row, a.target64) : -1;
  __syncthreads();  // also orders the stores above before the ones below
  auto put = [&](int i, float p, bool is_y) {
    const float v = T::load(z[i]);
    const float q = ci == 0.f ? 0.f : ci * exp2f((v - m) * c);
    float d = q - p;
    if (a.hard > 0) d += h1 * exp2f((v - m) * c1) - (is_y ? (float)a.hard : 0.f);
    dz[i] = T::store(g * d);
  };
  if (cls >= 0) {
    float p = 0;  // a class that is named twice has both entries' share
    for (int j = 0; j < a.k; ++j) p += cls_s[j] == cls ? p_s[j] : 0.f;
    put(cls, p, cls == y);
  }
  if (tid == 0 && y >= 0) {
    bool named = false;
    for (int j = 0; j < a.k; ++j) named = named || cls_s[j] == y;
    if (!named) {
      const float v = T::load(z[y]);
      float d = co == 0.f ? 0.f : co * exp2f((v - ref) * c);
      if (two) d += h1 * exp2f((v - m) * c1);
      dz[y] = T::store(g * (d - (float)a.hard));
    }
  }
}

void check_distill(const DistillArgs& a) {
  MX_CHECK(a.rows >= 0 && a.rows < (1ll << 31) && a.V >= 1 && a.V <= (1 << 30) && a.k >= 1 && a.k <= kTopMax,
           "distill_loss: bad sizes");
  MX_CHECK(a.temperature > 0 && a.hard >= 0 && a.hard <= 1 && (a.hard == 0 || a.target), "distill_loss: bad weights");
}

}  // namespace

void top_logits(const void* z, int type, int64_t ldz, int64_t rows, int V, int k, double temperature, void* values,
                int32_t* index, float* lse, hipStream_t st) {
  MX_CHECK(rows >= 0 && rows < (1ll << 31) && V >= 1 && V <= (1 << 30) && k >= 1 && k <= kTopMax && k <= V &&
               temperature > 0,
           "top_logits: bad sizes");
  if (rows == 0) return;
  MX_BY_TYPE(type, T, MX_LAUNCH(top_logits_k<T>, dim3((uint32_t)rows), dim3(kT), 0, st,
                                static_cast<const typename T::store_t*>(z), ldz, V, k, (float)(kLog2e / temperature),
                                (float)(1.0 / temperature), static_cast<typename T::store_t*>(values), index, lse));
}

void distill_fwd(const DistillArgs& a, float* loss_rows, float* loss, bool mean, hipStream_t st) {
  check_distill(a);
  if (a.rows > 0)
    MX_BY_TYPE(a.type, T, MX_LAUNCH(distill_fwd_k<T>, dim3((uint32_t)a.rows), dim3(kT), 0, st, a, loss_rows));
  if (loss) MX_LAUNCH(distill_mean_k, dim3(1), dim3(kT), 0, st, loss_rows, a.stats, a.rows, mean ? 1 : 0, loss);
}

void distill_bwd(const DistillArgs& a, const float* dloss, bool per_row, void* dz, hipStream_t st) {
  check_distill(a);
  if (a.rows > 0)
    MX_BY_TYPE(a.type, T, MX_LAUNCH(distill_bwd_k<T>, dim3((uint32_t)a.rows), dim3(kT), 0, st, a, dloss,
                                    per_row ? 1 : 0, static_cast<typename T::store_t*>(dz)));
}

}  // namespace mx
