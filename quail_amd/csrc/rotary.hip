// Rotary positions of q and k rows, any position, half or interleaved pairs,
// the whole head or its first part.
#include "qx_common.h"
#include "qx_status.h"

namespace qx {
namespace {

constexpr int kMaxPairs = 256;  // pairs of a head, in a wave's LDS
constexpr int kWaves = 4;       // rows per workgroup

struct RotaryArgs {
  const void *q, *k;
  void *qo, *ko;
  int64_t q_ld, k_ld, qo_ld, ko_ld;
  const int64_t* positions;
  const double* turns;  // of a pair, per position
  int64_t n;
  int HQ, heads, D, R;
  float factor;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T x[N];
};

__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(float v) { return v; }

template <int N, typename T>
__device__ __forceinline__ Pack<T, N> load(const T* x) {
  return *reinterpret_cast<const Pack<T, N>*>(x);
}

template <typename T, int N>
__device__ __forceinline__ void store(T* y, const Pack<T, N>& v) {
  *reinterpret_cast<Pack<T, N>*>(y) = v;
}

// N results in T, each rounded once (to nearest even)
template <int N>
__device__ __forceinline__ Pack<uint16_t, N> rounded(const float (&v)[N], const uint16_t*) {
  if constexpr (N == 1) {
    return {{f32_to_bf16(v[0])}};
  } else {
    Pack<uint32_t, N / 2> w;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w.x[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
    return __builtin_bit_cast(Pack<uint16_t, N>, w);
  }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> rounded(const float (&v)[N], const T*) {
  Pack<T, N> w;
#pragma unroll
  for (int i = 0; i < N; ++i) w.x[i] = (T)v[i];
  return w;
}

// y_a = a cos t - b sin t, y_b = b cos t + a sin t for each pair (a, b) of a
// head, t = position * frequency of the pair, cos and sin times `factor`.
// The position's turns are formed in 64 bits and their whole part dropped
// there. The frequency in turns and the product are rounded, so the angle is off by
// at most 3 2^-53 of itself: below what fp32 does to cos and sin (2^-22 of their
// pair) up to positions of some 2^29, and growing with the position past that
// (2^-12 at 2^40); past 2^53 the position itself is rounded. A row of cos and sin
// serves every head of q and k.
// A wave per row: its lanes compute the row's cos and sin into LDS, then take
// units of N pairs' elements (16 bytes; N = 1: rows whose strides, alignment or
// pairs do not allow that). Reads and writes each row once and is bound by HBM:
// 32 query and 8 key heads of 128 in 2 bytes, 15,654 rows 64 us from memory (321 MB
// at 5.0 TB/s; a copy reaches 5.1), 56 over and over. Waves enough hide the loads:
// with two units of a lane in flight 57, three 60, five 62-67. Stores past the
// caches 50, but what reads the rows next lost more (4000 rows and a copy of q 28.0
// us, 24.8 so). With N = 1 the pack takes 154 us (20 of 128 columns): 2 bytes a lane,
// and the columns that are only copied go by the same units, a division each.
template <typename T, int N, bool INTERLEAVED>
__global__ __launch_bounds__(64 * kWaves) void rotary_kernel(RotaryArgs p) {
  __shared__ float cs[kWaves][2][kMaxPairs];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * kWaves + wave;
  const int pairs = p.R / 2;
  if (row < p.n) {
    const double position = (double)p.positions[row];
    for (int i = lane; i < pairs; i += 64) {
      const double t = position * p.turns[i];
      float s, c;
      sincospif(2.0f * (float)(t - rint(t)), &s, &c);
      cs[wave][0][i] = c * p.factor;
      cs[wave][1][i] = s * p.factor;
    }
  }
  __syncthreads();
  if (row >= p.n) return;
  const T* q = static_cast<const T*>(p.q) + row * p.q_ld;
  const T* k = static_cast<const T*>(p.k) + row * p.k_ld;
  T* qo = static_cast<T*>(p.qo) + row * p.qo_ld;
  T* ko = static_cast<T*>(p.ko) + row * p.ko_ld;
  auto in = [&](int head) { return head < p.HQ ? q + head * p.D : k + (head - p.HQ) * p.D; };
  auto out = [&](int head) { return head < p.HQ ? qo + head * p.D : ko + (head - p.HQ) * p.D; };
  // a unit: N pairs of half layout (two packs), or the 2 N elements of N
  // interleaved ones
  const int units = pairs / N;
  const int step_h = 64 / units, step_u = 64 % units;
  int head = lane / units, u = lane % units;
  while (head < p.heads) {
    const int at_a = INTERLEAVED ? 2 * u * N : u * N, at_b = INTERLEAVED ? at_a + N : at_a + pairs;
    const Pack<T, N> a = load<N>(in(head) + at_a), b = load<N>(in(head) + at_b);
    const float *c = &cs[wave][0][u * N], *s = &cs[wave][1][u * N];
    float xa[N], xb[N];
    if constexpr (!INTERLEAVED || N == 1) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float va = to_f32(a.x[e]), vb = to_f32(b.x[e]);
        xa[e] = va * c[e] - vb * s[e];
        xb[e] = vb * c[e] + va * s[e];
      }
    } else {  // each pack holds N / 2 pairs
      auto turn = [&](const Pack<T, N>& v, float (&y)[N], int first) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const float va = to_f32(v.x[2 * e]), vb = to_f32(v.x[2 * e + 1]);
          y[2 * e] = va * c[first + e] - vb * s[first + e];
          y[2 * e + 1] = vb * c[first + e] + va * s[first + e];
        }
      };
      turn(a, xa, 0);
      turn(b, xb, N / 2);
    }
    store(out(head) + at_a, rounded(xa, (T*)nullptr));
    store(out(head) + at_b, rounded(xb, (T*)nullptr));
    head += step_h;
    u += step_u;
    if (u >= units) {
      u -= units;
      ++head;
    }
  }
  // the rest of each head as it is
  const int rest = (p.D - p.R) / N;
  if (rest == 0) return;
  for (int i = lane; i < p.heads * rest; i += 64) {
    const int h = i / rest, e = p.R + i % rest * N;
    const T *x = in(h) + e;
    T* y = out(h) + e;
    if (x != y) store(y, load<N>(x));
  }
}

template <typename T>
int launch(const RotaryArgs& a, bool interleaved, hipStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.qo | (uintptr_t)(a.k ? a.k : a.q) |
                       (uintptr_t)(a.ko ? a.ko : a.qo);
  const bool wide = (at & 15) == 0 && (a.q_ld | a.k_ld | a.qo_ld | a.ko_ld) % N == 0 &&
                    (a.R / 2) % N == 0 && a.D % N == 0;
  const dim3 grid((unsigned)((a.n + kWaves - 1) / kWaves)), block(64 * kWaves);
#define QX_ROTARY(NN, I) \
  hipLaunchKernelGGL((rotary_kernel<T, NN, I>), grid, block, 0, stream, a)
  if (wide) {
    if (interleaved) QX_ROTARY(N, true); else QX_ROTARY(N, false);
  } else {
    if (interleaved) QX_ROTARY(1, true); else QX_ROTARY(1, false);
  }
#undef QX_ROTARY
  QX_LAUNCH_STATUS();
}

}  // namespace
}  // namespace qx

using namespace qx;

extern "C" {

int qx_rotary(const void* q, int64_t q_ld, const void* k, int64_t k_ld, void* q_out,
              int64_t qo_ld, void* k_out, int64_t ko_ld, const int64_t* positions,
              const double* turns, float factor, int64_t n, int64_t HQ, int64_t HK, int64_t D,
              int64_t rotary_dim, int interleaved, int type, hipStream_t stream) {
  QX_CHECK(n >= 0 && HQ >= 0 && HK >= 0 && HQ + HK > 0, "rotary: %lld rows of %lld and %lld heads",
           (long long)n, (long long)HQ, (long long)HK);
  QX_CHECK(n == 0 || (positions && turns && (HQ == 0 || (q && q_out)) && (HK == 0 || (k && k_out))),
           "rotary: null pointer");
  QX_CHECK(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= D && rotary_dim <= 2 * kMaxPairs,
           "rotary: %lld columns of a head of %lld (an even number, at most %d)",
           (long long)rotary_dim, (long long)D, 2 * kMaxPairs);
  QX_CHECK(type >= 0 && type <= 2, "rotary: type %d (0 bf16, 1 fp16, 2 fp32)", type);
  QX_CHECK(D <= 65536 && HQ + HK <= 65536 && (HQ + HK) * D < (1LL << 30) && n < (1LL << 26),
           "rotary: %lld rows of %lld heads exceed one launch", (long long)n, (long long)(HQ + HK));
  QX_CHECK((HQ == 0 || (q_ld >= HQ * D && qo_ld >= HQ * D)) &&
               (HK == 0 || (k_ld >= HK * D && ko_ld >= HK * D)),
           "rotary: rows that overlap");
  if (n == 0) return QX_OK;
  RotaryArgs a{q, k, q_out, k_out, q_ld, k_ld, qo_ld, ko_ld, positions, turns, n, (int)HQ,
               (int)(HQ + HK), (int)D, (int)rotary_dim, factor};
  if (HQ == 0) a.q = a.k, a.qo = a.ko, a.q_ld = k_ld, a.qo_ld = ko_ld;
  if (HK == 0) a.k = a.q, a.ko = a.qo, a.k_ld = q_ld, a.ko_ld = qo_ld;
  return type == 0 ? launch<uint16_t>(a, interleaved, stream)
                   : type == 1 ? launch<_Float16>(a, interleaved, stream)
                               : launch<float>(a, interleaved, stream);
}

}  // extern "C"
