// Qwen3's q-norm and RoPE on a wave's query rows as the attention kernels load
// them (32x32 MFMA operand layout, D = 128).
#pragma once

#include "qx_common.h"

namespace qx {

// QN != 0: q holds the raw (pre-norm) q columns of the qkv projection, and
// the kernel applies each row's qk-norm and RoPE as it loads it: position
// pos[row], the cos/sin cache cs ((max_pos, 128) [cos | sin], bf16 for
// QN = 1, fp32 for QN = 2), the q-norm weight qw and eps.
struct QNormArgs {
  const int64_t* pos;
  const void* cs;       // (positions, 128) cos | sin; bf16 (QN 1) or fp32 (QN 2)
  const uint16_t* qw;  // the q-norm weight (128), bf16
  float eps;
};

// What q-norm on load reads for one lane: the q-norm weight of its 64
// columns (c*16 + half*8 + k, c, k < 8), then, once the row's position is
// in, the row's cos / sin of its first-half columns (bf16 for QN = 1, fp32
// for QN = 2), raw as loaded.
template <int QN>
struct QNormIn {
  static constexpr int kCs = QN == 2 ? 16 : 8;
  uint4 wq[8];
  uint4 cs[kCs];
};

template <int QN>
__device__ __forceinline__ void q_norm_load_weights(QNormIn<QN>& in, const QNormArgs& qn,
                                                    int half) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    in.wq[c] = *reinterpret_cast<const uint4*>(qn.qw + c * 16 + half * 8);
}

template <int QN>
__device__ __forceinline__ void q_norm_load_row(QNormIn<QN>& in, const QNormArgs& qn, int64_t p,
                                                int half) {
  if constexpr (QN == 1) {
    const uint16_t* row_cs = reinterpret_cast<const uint16_t*>(qn.cs) + p * 128;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      in.cs[2 * c] = *reinterpret_cast<const uint4*>(row_cs + c * 16 + half * 8);
      in.cs[2 * c + 1] = *reinterpret_cast<const uint4*>(row_cs + 64 + c * 16 + half * 8);
    }
  } else {
    const float* row_cs = reinterpret_cast<const float*>(qn.cs) + p * 128;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        in.cs[4 * c + 2 * e] = *reinterpret_cast<const uint4*>(row_cs + c * 16 + half * 8 + e * 4);
        in.cs[4 * c + 2 * e + 1] =
            *reinterpret_cast<const uint4*>(row_cs + 64 + c * 16 + half * 8 + e * 4);
      }
  }
}

// The lane's 64 q columns of one head through qk-norm and RoPE with the
// qk-norm-rope pass's arithmetic and summation tree. The pass sums a head's
// 16 column groups j (columns 4j.. and 64 + 4j..) with a butterfly over j
// (xor 8, 4, 2, 1); group j = 4c + 2 half + e (c < 4) is this lane's
// columns c*16 + half*8 + 4e.., so the xor-8 and xor-4 levels pair the
// lane's own groups (c ^ 2, c ^ 1), xor 2 pairs it with lane ^ 32 and xor 1
// its own e ^ 1: the same sums of the same terms, and each addition
// commutes, so the rows come out bit for bit as the pass writes them.
template <int QN>
__device__ __forceinline__ void q_norm_rope_apply(v8s (&qf)[8], const QNormIn<QN>& in,
                                                  float eps) {
  float cosv[4][2][4], sinv[4][2][4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if constexpr (QN == 1) {
      const uint4 cw = in.cs[2 * c], sw = in.cs[2 * c + 1];
      bf16x4_to_f32(make_uint2(cw.x, cw.y), cosv[c][0]);
      bf16x4_to_f32(make_uint2(cw.z, cw.w), cosv[c][1]);
      bf16x4_to_f32(make_uint2(sw.x, sw.y), sinv[c][0]);
      bf16x4_to_f32(make_uint2(sw.z, sw.w), sinv[c][1]);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 cv = in.cs[4 * c + 2 * e], sv = in.cs[4 * c + 2 * e + 1];
        cosv[c][e][0] = __uint_as_float(cv.x); cosv[c][e][1] = __uint_as_float(cv.y);
        cosv[c][e][2] = __uint_as_float(cv.z); cosv[c][e][3] = __uint_as_float(cv.w);
        sinv[c][e][0] = __uint_as_float(sv.x); sinv[c][e][1] = __uint_as_float(sv.y);
        sinv[c][e][2] = __uint_as_float(sv.z); sinv[c][e][3] = __uint_as_float(sv.w);
      }
    }
  }
  auto group = [&](const v8s& x, int e, float (&out)[4]) {
    const uint4 w = __builtin_bit_cast(uint4, x);
    bf16x4_to_f32(e ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y), out);
  };
  float s[4][2];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float a[4], b[4];
      group(qf[c], e, a);
      group(qf[c + 4], e, b);
      s[c][e] = norm_part4(a, b);
    }
  float w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) w[e] = sum_halves((s[0][e] + s[2][e]) + (s[1][e] + s[3][e]));
  const float rstd = norm_rstd<128>(w[0] + w[1], eps);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint4 lo = __builtin_bit_cast(uint4, qf[c]), hi = __builtin_bit_cast(uint4, qf[c + 4]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float a[4], b[4], wa[4], wb[4], oa[4], ob[4];
      group(qf[c], e, a);
      group(qf[c + 4], e, b);
      group(__builtin_bit_cast(v8s, in.wq[c]), e, wa);
      group(__builtin_bit_cast(v8s, in.wq[c + 4]), e, wb);
      norm_rope4(a, b, wa, wb, cosv[c][e], sinv[c][e], rstd, oa, ob);
      const uint32_t o0 = pack2_bf16(oa[0], oa[1]), o1 = pack2_bf16(oa[2], oa[3]);
      const uint32_t p0 = pack2_bf16(ob[0], ob[1]), p1 = pack2_bf16(ob[2], ob[3]);
      if (e) {
        lo.z = o0; lo.w = o1; hi.z = p0; hi.w = p1;
      } else {
        lo.x = o0; lo.y = o1; hi.x = p0; hi.y = p1;
      }
    }
    qf[c] = __builtin_bit_cast(v8s, lo);
    qf[c + 4] = __builtin_bit_cast(v8s, hi);
  }
}

}  // namespace qx
