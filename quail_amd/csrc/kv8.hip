// The 8-bit KV arena's writes, and copies of whole pages of any arena.
//
// An 8-bit pool holds e4m3 codes, (pages * 16, HK, D) bytes, K and V apart,
// and one power-of-two scale per (page, KV head), an E8M0 byte b that stands
// for 2^(b - 127), at scales[(page * HK + head) * 2 + (0 for K, 1 for V)].
#include <algorithm>
#include <new>
#include <vector>

#include "qx_common.h"
#include "qx_status.h"

namespace qx {
namespace {

constexpr int kPage = 16;  // tokens per arena page
constexpr float kF32Max = 3.402823466e38f;

// The E8M0 byte of the least power of two s with amax <= 448 s, at least 1:
// with amax = 1.m * 2^e that is 2^(e - 8), and twice that where 1.m > 1.75.
// Adding the distance from the fraction of 1.75 to the next power of two
// carries into the exponent exactly where the fraction is past it.
__device__ __forceinline__ int scale_byte(float amax) {
  return max((int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8, 1);
}

// Infinities count as the largest finite value (e4m3 has none); NaN stays.
__device__ __forceinline__ float finite(float x) {
  return x != x ? x : fminf(fmaxf(x, -kF32Max), kF32Max);
}

__device__ __forceinline__ uint32_t scaled4(const float* x, int shift) {
  return pack4_fp8(__builtin_ldexpf(x[0], shift), __builtin_ldexpf(x[1], shift),
                   __builtin_ldexpf(x[2], shift), __builtin_ldexpf(x[3], shift));
}

// One page of one head per wave. Item i of `items` is (destination page,
// source page, kept rows, first row, rows): the page's rows [0, keep) are
// the source page's, the next `count` are fresh rows row0, row0 + 1, ...; the
// rest of the page stays as it is. The scale is the fresh rows' own, or the
// larger of that and the source page's where rows are kept: the kept codes
// then move by a power of two, exactly unless they become subnormal.
// Waves of an item: HK of K, HK of V, then (QKV, with a q output) HQ of q.
// QKV: rows are the qkv projection's; q and K go through their norm and RoPE
// (norm_rope4) and K from fp32 to its code in one rounding. Otherwise k and
// v are rows as the pool takes them.
// Streams 2 * (2 HK + HQ) * D bytes a row in and (2 HK + 2 HQ) * D out; a
// wave holds its 16 x D values in registers between the maximum and the codes.
struct WriteArgs {
  const uint16_t *x, *v;  // qkv rows, or K rows and V rows
  int64_t x_ld, v_ld;
  uint16_t* qo;
  int64_t qo_ld;
  uint8_t *kp, *vp, *scales;
  const int* items;
  const void* cs;
  const int64_t* pos;
  const uint16_t *qw, *kw;
  float eps;
  int64_t waves;
  int slots, HQ, HK;
};

template <int D, bool QKV, bool CS_F32>
__global__ __launch_bounds__(256) void kv8_write_kernel(WriteArgs p) {
  constexpr int LPR = D / 8;         // lanes per row, 8 columns each
  constexpr int RPP = 64 / LPR;      // rows per pass
  constexpr int PASSES = kPage / RPP;
  constexpr int HALF = D / 2;
  const int lane = threadIdx.x & 63;
  const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wid >= p.waves) return;
  const int slot = (int)(wid % p.slots);
  const int* item = p.items + wid / p.slots * 5;
  const int dst = item[0], src = item[1], keep = item[2], row0 = item[3], count = item[4];
  const bool is_v = slot >= p.HK && slot < 2 * p.HK;
  const bool is_q = QKV && slot >= 2 * p.HK;
  const bool rotate = QKV && !is_v;
  const int head = is_q ? slot - 2 * p.HK : is_v ? slot - p.HK : slot;
  const int j = lane % LPR;
  // this lane's columns: [c0, c0 + 4) and [c1, c1 + 4)
  const int c0 = rotate ? 4 * j : 8 * j, c1 = rotate ? HALF + 4 * j : 8 * j + 4;
  const uint16_t* x = QKV || !is_v ? p.x : p.v;
  const int64_t x_ld = QKV || !is_v ? p.x_ld : p.v_ld;
  const int64_t col = (int64_t)D * (!QKV ? head : is_q ? head : is_v ? p.HQ + p.HK + head
                                                                     : p.HQ + head);
  float wa[4], wb[4];
  if (rotate) {
    const uint16_t* w = is_q ? p.qw : p.kw;
    bf16x4_to_f32(*reinterpret_cast<const uint2*>(w + c0), wa);
    bf16x4_to_f32(*reinterpret_cast<const uint2*>(w + c1), wb);
  }
  uint8_t* pool = is_v ? p.vp : p.kp;
  const int64_t kv_row = (int64_t)p.HK * D;
  const int side = is_v ? 1 : 0;
  int b_old = 0;
  if (!is_q && keep > 0) b_old = p.scales[((int64_t)src * p.HK + head) * 2 + side];
  float y[PASSES][8];
  float amax = 0.f;
#pragma unroll
  for (int t = 0; t < PASSES; ++t) {
    const int r = t * RPP + lane / LPR;  // row of the page
    const bool fresh = r >= keep && r < keep + count;
    float a[4] = {}, b[4] = {};
    if (fresh) {
      const int64_t row = (int64_t)row0 + r - keep;
      const uint16_t* xr = x + row * x_ld + col;
      bf16x4_to_f32(*reinterpret_cast<const uint2*>(xr + c0), a);
      bf16x4_to_f32(*reinterpret_cast<const uint2*>(xr + c1), b);
    }
    if (rotate) {
      // a row's lanes are all fresh or all not: the sum stays inside them
      const float rstd = norm_rstd<D>(group_sum<LPR>(norm_part4(a, b)), p.eps);
      if (fresh) {
        const int64_t row = (int64_t)row0 + r - keep;
        float cosv[4], sinv[4], oa[4], ob[4];
        const int64_t at = p.pos[row] * D;
        if (CS_F32) {
          const float* c = reinterpret_cast<const float*>(p.cs) + at;
          const float4 c4 = *reinterpret_cast<const float4*>(c + c0);
          const float4 s4 = *reinterpret_cast<const float4*>(c + c1);
          cosv[0] = c4.x; cosv[1] = c4.y; cosv[2] = c4.z; cosv[3] = c4.w;
          sinv[0] = s4.x; sinv[1] = s4.y; sinv[2] = s4.z; sinv[3] = s4.w;
        } else {
          const uint16_t* c = reinterpret_cast<const uint16_t*>(p.cs) + at;
          bf16x4_to_f32(*reinterpret_cast<const uint2*>(c + c0), cosv);
          bf16x4_to_f32(*reinterpret_cast<const uint2*>(c + c1), sinv);
        }
        norm_rope4(a, b, wa, wb, cosv, sinv, rstd, oa, ob);
        if (is_q) {
          uint16_t* out = p.qo + row * p.qo_ld + head * D;
          *reinterpret_cast<uint2*>(out + c0) =
              make_uint2(pack2_bf16(oa[0], oa[1]), pack2_bf16(oa[2], oa[3]));
          *reinterpret_cast<uint2*>(out + c1) =
              make_uint2(pack2_bf16(ob[0], ob[1]), pack2_bf16(ob[2], ob[3]));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          a[k] = oa[k];
          b[k] = ob[k];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      y[t][k] = finite(a[k]);
      y[t][4 + k] = finite(b[k]);
      amax = fmaxf(amax, fmaxf(fabsf(y[t][k]), fabsf(y[t][4 + k])));
    }
  }
  if (is_q) return;
  amax = group_max<64>(amax);
  const int need = scale_byte(amax);
  const int b = keep > 0 ? max(b_old, need) : need;
  const bool move = src != dst || b != b_old;  // the kept rows change
#pragma unroll
  for (int t = 0; t < PASSES; ++t) {
    const int r = t * RPP + lane / LPR;
    uint8_t* out = pool + ((int64_t)dst * kPage + r) * kv_row + head * D;
    if (r < keep) {
      if (!move) continue;
      const uint8_t* in = pool + ((int64_t)src * kPage + r) * kv_row + head * D;
      const int lo = *reinterpret_cast<const int*>(in + c0);
      const int hi = *reinterpret_cast<const int*>(in + c1);
      const float old[8] = {
          __builtin_amdgcn_cvt_f32_fp8(lo, 0), __builtin_amdgcn_cvt_f32_fp8(lo, 1),
          __builtin_amdgcn_cvt_f32_fp8(lo, 2), __builtin_amdgcn_cvt_f32_fp8(lo, 3),
          __builtin_amdgcn_cvt_f32_fp8(hi, 0), __builtin_amdgcn_cvt_f32_fp8(hi, 1),
          __builtin_amdgcn_cvt_f32_fp8(hi, 2), __builtin_amdgcn_cvt_f32_fp8(hi, 3)};
      *reinterpret_cast<uint32_t*>(out + c0) = scaled4(old, b_old - b);
      *reinterpret_cast<uint32_t*>(out + c1) = scaled4(old + 4, b_old - b);
    } else if (r < keep + count) {
      *reinterpret_cast<uint32_t*>(out + c0) = scaled4(y[t], 127 - b);
      *reinterpret_cast<uint32_t*>(out + c1) = scaled4(y[t] + 4, 127 - b);
    }
  }
  if (lane == 0) p.scales[((int64_t)dst * p.HK + head) * 2 + side] = (uint8_t)b;
}

int kv8_write_launch(WriteArgs& a, bool qkv, int64_t n_items, int64_t HK, int64_t D, int cs_is_f32,
                     hipStream_t stream) {
  QX_CHECK(D == 64 || D == 128, "kv8_write: head_dim %lld (64 or 128)", (long long)D);
  QX_CHECK(HK > 0 && n_items >= 0, "kv8_write: heads %lld, items %lld", (long long)HK,
           (long long)n_items);
  if (n_items == 0) return QX_OK;
  a.waves = n_items * a.slots;
  QX_CHECK(a.waves <= (1LL << 26) - 4, "kv8_write: %lld items of %d heads exceed one launch",
           (long long)n_items, a.slots);  // 2^32 threads
  const dim3 grid((unsigned)((a.waves + 3) / 4)), block(256);
#define QX_KV8(DD, Q, F) hipLaunchKernelGGL((kv8_write_kernel<DD, Q, F>), grid, block, 0, stream, a)
  if (!qkv) {
    if (D == 128) QX_KV8(128, false, false); else QX_KV8(64, false, false);
  } else if (cs_is_f32) {
    if (D == 128) QX_KV8(128, true, true); else QX_KV8(64, true, true);
  } else {
    if (D == 128) QX_KV8(128, true, false); else QX_KV8(64, true, false);
  }
#undef QX_KV8
  QX_LAUNCH_STATUS();
}

// Pages src[i] -> dst[i] of every pool: the page ids travel in the kernel's
// arguments, so a copy needs no upload and nothing of the caller's stays in
// use after the call.
constexpr int kCopyIds = 440;
struct CopyIds {
  int src[kCopyIds], dst[kCopyIds];
};
struct CopyRegion {
  uint8_t* base;
  int64_t pool_stride, page_bytes;
  int pools;
};

// blockIdx.x: page of the list; blockIdx.y: pool (the codes' pools, then the
// scales'); blockIdx.z: part of the page.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyRegion big, CopyRegion small,
                                                         CopyIds ids) {
  const int pool = blockIdx.y;
  const bool tail = pool >= big.pools;
  if (tail && blockIdx.z) return;
  const CopyRegion r = tail ? small : big;
  uint8_t* at = r.base + (tail ? pool - big.pools : pool) * r.pool_stride;
  const uint8_t* s = at + ids.src[blockIdx.x] * r.page_bytes;
  uint8_t* d = at + ids.dst[blockIdx.x] * r.page_bytes;
  if (tail) {
    for (int64_t c = threadIdx.x; c < r.page_bytes / 2; c += 256)
      reinterpret_cast<uint16_t*>(d)[c] = reinterpret_cast<const uint16_t*>(s)[c];
    return;
  }
  const int64_t chunks = r.page_bytes / 16;
  for (int64_t c = blockIdx.z * 256 + threadIdx.x; c < chunks; c += 256 * gridDim.z)
    reinterpret_cast<uint4*>(d)[c] = reinterpret_cast<const uint4*>(s)[c];
}

bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace
}  // namespace qx

using namespace qx;

extern "C" {

int qx_qk_norm_rope_kv8(const void* qkv, int64_t qkv_ld, void* q_out, int64_t q_ld, void* k_pool,
                        void* v_pool, void* scales, const int* items, int64_t n_items,
                        const void* cos_sin, int cs_is_f32, const int64_t* positions,
                        const void* q_w, const void* k_w, int64_t HQ, int64_t HK, int64_t D,
                        float eps, hipStream_t stream) {
  QX_CHECK(qkv && k_pool && v_pool && scales && cos_sin && positions && q_w && k_w &&
               (items || n_items == 0),
           "qk_norm_rope_kv8: null pointer");
  QX_CHECK(HQ > 0, "qk_norm_rope_kv8: heads");
  QX_CHECK(qkv_ld % 4 == 0 && q_ld % 4 == 0 && aligned(qkv, 8) && aligned(q_out, 8) &&
               aligned(k_pool, 4) && aligned(v_pool, 4) && aligned(cos_sin, 16) &&
               aligned(q_w, 8) && aligned(k_w, 8),
           "qk_norm_rope_kv8: strides or alignment");
  WriteArgs a{(const uint16_t*)qkv, nullptr, qkv_ld, 0, (uint16_t*)q_out, q_ld,
              (uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)scales, items, cos_sin, positions,
              (const uint16_t*)q_w, (const uint16_t*)k_w, eps, 0,
              (int)(2 * HK + (q_out ? HQ : 0)), (int)HQ, (int)HK};
  return kv8_write_launch(a, true, n_items, HK, D, cs_is_f32, stream);
}

int qx_kv8_write(const void* k, int64_t k_ld, const void* v, int64_t v_ld, void* k_pool,
                 void* v_pool, void* scales, const int* items, int64_t n_items, int64_t HK,
                 int64_t D, hipStream_t stream) {
  QX_CHECK(k && v && k_pool && v_pool && scales && (items || n_items == 0),
           "kv8_write: null pointer");
  QX_CHECK(k_ld % 4 == 0 && v_ld % 4 == 0 && aligned(k, 8) && aligned(v, 8) &&
               aligned(k_pool, 4) && aligned(v_pool, 4),
           "kv8_write: strides or alignment");
  WriteArgs a{(const uint16_t*)k, (const uint16_t*)v, k_ld, v_ld, nullptr, 0,
              (uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)scales, items, nullptr, nullptr,
              nullptr, nullptr, 0.f, 0, (int)(2 * HK), 0, (int)HK};
  return kv8_write_launch(a, false, n_items, HK, D, 0, stream);
}

static int copy_pages(void* pools, int64_t n_pools, int64_t pool_stride, int64_t page_bytes,
                      void* scales, int64_t n_scale_pools, int64_t scale_stride,
                      int64_t scale_bytes, const int* src, const int* dst, int64_t count,
                      int64_t num_pages, hipStream_t stream) {
  QX_CHECK(pools && (scales || n_scale_pools == 0) && (count == 0 || (src && dst)),
           "copy_pages: null pointer");
  QX_CHECK(n_pools > 0 && n_scale_pools >= 0 && n_pools + n_scale_pools < 65536 && count >= 0 &&
               num_pages >= 0,
           "copy_pages: %lld + %lld pools, %lld pages", (long long)n_pools,
           (long long)n_scale_pools, (long long)count);
  QX_CHECK(page_bytes > 0 && page_bytes % 16 == 0 && pool_stride % 16 == 0 && aligned(pools, 16) &&
               (n_scale_pools == 0 || (scale_bytes > 0 && scale_bytes % 2 == 0 &&
                                       scale_stride % 2 == 0 && aligned(scales, 2))),
           "copy_pages: page sizes or alignment");
  std::vector<uint8_t> role(num_pages, 0);  // 1: a source, 2: a destination
  for (int64_t i = 0; i < count; ++i) {
    QX_CHECK(src[i] >= 0 && src[i] < num_pages && dst[i] >= 0 && dst[i] < num_pages,
             "copy_pages: page %d -> %d of %lld", src[i], dst[i], (long long)num_pages);
    QX_CHECK(!(role[src[i]] & 2), "copy_pages: page %d is a source and a destination", src[i]);
    QX_CHECK(!role[dst[i]], "copy_pages: page %d is a destination twice, or also a source",
             dst[i]);
    if (src[i] == dst[i]) QX_CHECK(false, "copy_pages: page %d onto itself", src[i]);
    role[src[i]] = 1;
    role[dst[i]] = 2;
  }
  const CopyRegion big{(uint8_t*)pools, pool_stride, page_bytes, (int)n_pools};
  const CopyRegion small{(uint8_t*)scales, scale_stride, scale_bytes, (int)n_scale_pools};
  for (int64_t first = 0; first < count; first += kCopyIds) {
    CopyIds ids;
    const int n = (int)std::min<int64_t>(kCopyIds, count - first);
    for (int i = 0; i < n; ++i) {
      ids.src[i] = src[first + i];
      ids.dst[i] = dst[first + i];
    }
    const int64_t parts = std::min<int64_t>((page_bytes / 16 + 1023) / 1024, 64);
    hipLaunchKernelGGL(copy_pages_kernel,
                       dim3((unsigned)n, (unsigned)(n_pools + n_scale_pools), (unsigned)parts),
                       dim3(256), 0, stream, big, small, ids);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return QX_OK;
}

int qx_copy_pages(void* pools, int64_t n_pools, int64_t pool_stride, int64_t page_bytes,
                  void* scales, int64_t n_scale_pools, int64_t scale_stride, int64_t scale_bytes,
                  const int* src, const int* dst, int64_t count, int64_t num_pages,
                  hipStream_t stream) {
  try {
    return copy_pages(pools, n_pools, pool_stride, page_bytes, scales, n_scale_pools,
                      scale_stride, scale_bytes, src, dst, count, num_pages, stream);
  } catch (const std::bad_alloc&) {
    qx::set_error("copy_pages: out of host memory");
    return QX_EINVAL;
  }
}

}  // extern "C"
