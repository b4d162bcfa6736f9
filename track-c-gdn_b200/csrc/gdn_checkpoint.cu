// gdn_checkpoint.cu -- activations to int8 groups and back (format in
// gdn_recurrence.cuh: 128 values of a row share one power of two).
//
// A warp takes kItems groups of one tensor, loads them all before it works on
// the first, finds each group's largest magnitude with one warp reduction, and
// writes a byte a value and a byte a group: 3 bytes a value each way for 2-byte
// types, bound by HBM.  Where a tensor's groups follow one another in memory
// (full groups, rows without gaps) a group's place is its number; elsewhere it
// takes two 32-bit divisions a group.  134 M bf16 values: 60 us each way at 6.7
// TB/s, as fast as a copy.
#include "gdn_recurrence.cuh"

namespace gdn {
namespace rec {

constexpr int kPackTensors = 4;  // tensors of one launch
constexpr int kItems = 8;

struct PackTensor {
  void *data;        // pack: the input; unpack: the output [rows, cols]
  uint8_t *values;   // [rows, cols] int8
  uint8_t *scales;   // [rows, groups]
  int64_t outer_stride, inner_stride;  // row r lies at r / inner, r % inner
  int64_t cols;
  uint32_t inner, groups, items;
  uint32_t first;    // the tensor's first warp in the launch
  int flat;          // groups follow one another
};
struct Pack {
  PackTensor t[kPackTensors];
  int count;
};

// A group's elements, from the start of the data (as it lies) and of the values.
// (32-bit numbers: rows, columns and groups in all are below 2^31.)
struct Place {
  int64_t data, values;
  int left;  // values of the row from there on
};
__device__ __forceinline__ Place place_of(const PackTensor &t, uint32_t item, bool unpack) {
  if (t.flat) {
    const int64_t at = static_cast<int64_t>(item) * kGroupValues;
    return Place{at, at, kGroupValues};
  }
  const uint32_t row = item / t.groups, c0 = (item - row * t.groups) * kGroupValues;
  const int64_t values = row * t.cols + c0;
  const uint32_t outer = row / t.inner;
  return Place{unpack ? values : outer * t.outer_stride + (row - outer * t.inner) * t.inner_stride + c0, values,
               static_cast<int>(min(t.cols - c0, int64_t{kGroupValues}))};
}
__device__ __forceinline__ int tensor_of(const Pack &p, uint32_t warp) {
  int k = 0;
#pragma unroll
  for (int i = 1; i < kPackTensors; ++i) k = i < p.count && warp >= p.t[i].first ? i : k;
  return k;
}

// The largest magnitude of a lane's four values, as bits whose order is that of
// the values (16 bits, twice, for 2-byte types), and those bits as an fp32's.
__device__ __forceinline__ uint32_t lane_max(const Raw<__nv_bfloat16> &r) {
  const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162 *>(&r.v.x);
  const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162 *>(&r.v.y);
  const __nv_bfloat162 m = __hmax2_nan(__habs2(a), __habs2(b)), n = __hmax2_nan(m, __lowhigh2highlow(m));
  return *reinterpret_cast<const uint32_t *>(&n);
}
__device__ __forceinline__ uint32_t lane_max(const Raw<__half> &r) {
  const __half2 a = *reinterpret_cast<const __half2 *>(&r.v.x), b = *reinterpret_cast<const __half2 *>(&r.v.y);
  const __half2 m = __hmax2_nan(__habs2(a), __habs2(b)), n = __hmax2_nan(m, __lowhigh2highlow(m));
  return *reinterpret_cast<const uint32_t *>(&n);
}
__device__ __forceinline__ uint32_t lane_max(const Raw<float> &r) {
  return abs_max_bits(f2_pack(r.v.x, r.v.y), f2_pack(r.v.z, r.v.w));
}
template <typename E>
__device__ __forceinline__ uint32_t magnitude(uint32_t m) {
  if constexpr (std::is_same<E, float>::value) return m;
  if constexpr (std::is_same<E, __half>::value)
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(m))));
  return m << 16;
}

template <typename E, bool kVec>
__global__ void __launch_bounds__(kThreads) checkpoint_pack_kernel(const __grid_constant__ Pack p) {
  const int lane = threadIdx.x & 31;
  const uint32_t warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const PackTensor &t = p.t[tensor_of(p, warp)];
  const uint32_t item0 = (warp - t.first) * kItems;
  if (item0 >= t.items) return;
  const int n = static_cast<int>(min(t.items - item0, uint32_t{kItems}));
  Raw<E> raw[kItems];
  if (kVec && t.flat && n == kItems) {
    // groups one after the other; lane i works out the scale of group i
    const E *src = static_cast<const E *>(t.data) + static_cast<int64_t>(item0) * kGroupValues;
    uint32_t *dst = reinterpret_cast<uint32_t *>(t.values + static_cast<int64_t>(item0) * kGroupValues) + lane;
#pragma unroll
    for (int i = 0; i < kItems; ++i) raw[i] = load4<E, kVec>(src + i * kGroupValues, lane, kGroupValues);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, lane_max(raw[i]));
      top = lane == i ? m : top;
    }
    const uint32_t ex = group_exponent(magnitude<E>(top), exp_cap<E>());
    if (lane < kItems) t.scales[item0 + lane] = static_cast<uint8_t>(ex);
    if (__all_sync(0xffffffffu, ex < exp_cap<E>())) {
      const float inv = group_inverse(ex);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        uint64_t a, b;
        raw[i].pairs(a, b);
        const float f = __shfl_sync(0xffffffffu, inv, i);
        dst[i * (kGroupValues / 4)] = __byte_perm(quantise2(a, f), quantise2(b, f), 0x5410);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        uint64_t a, b;
        raw[i].pairs(a, b);
        dst[i * (kGroupValues / 4)] = quantise4(a, b, __shfl_sync(0xffffffffu, ex, i), exp_cap<E>());
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    raw[i] = {};
    if (i < n) {
      const Place at = place_of(t, item0 + i, false);
      raw[i] = load4<E, kVec>(static_cast<const E *>(t.data) + at.data, lane, at.left);
    }
  }
  uint32_t mine = 0;  // lane i: the exponent of group i
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (i >= n) break;
    const Place at = place_of(t, item0 + i, false);
    uint64_t a, b;
    raw[i].pairs(a, b);
    const uint32_t ex = group_exponent(__reduce_max_sync(0xffffffffu, abs_max_bits(a, b)), exp_cap<E>());
    const uint32_t q = quantise4(a, b, ex, exp_cap<E>());
    uint8_t *dst = t.values + at.values;
    if constexpr (kVec) {
      if (4 * lane < at.left) reinterpret_cast<uint32_t *>(dst)[lane] = q;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lane + 32 * j < at.left) dst[lane + 32 * j] = static_cast<uint8_t>(q >> (8 * j));
    }
    mine = lane == i ? ex : mine;
  }
  if (lane < n) t.scales[item0 + lane] = static_cast<uint8_t>(mine);
}

template <typename E, bool kVec>
__global__ void __launch_bounds__(kThreads) checkpoint_unpack_kernel(const __grid_constant__ Pack p) {
  const int lane = threadIdx.x & 31;
  const uint32_t warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const PackTensor &t = p.t[tensor_of(p, warp)];
  const uint32_t item0 = (warp - t.first) * kItems;
  if (item0 >= t.items) return;
  const int n = static_cast<int>(min(t.items - item0, uint32_t{kItems}));
  const uint32_t mine = lane < n ? __ldg(t.scales + item0 + lane) : 0;
  if (kVec && t.flat && n == kItems) {
    // groups one after the other: 8 values a lane, two groups a load
    const uint2 *src = reinterpret_cast<const uint2 *>(t.values + static_cast<int64_t>(item0) * kGroupValues) + lane;
    E *dst = static_cast<E *>(t.data) + static_cast<int64_t>(item0) * kGroupValues + 8 * lane;
    uint2 v[kItems / 2];
#pragma unroll
    for (int i = 0; i < kItems / 2; ++i) v[i] = __ldg(src + 32 * i);
#pragma unroll
    for (int i = 0; i < kItems / 2; ++i) {
      uint64_t a, b, c, d;
      const uint32_t ex = __shfl_sync(0xffffffffu, mine, 2 * i + (lane >> 4));
      dequantise4(v[i].x, ex, a, b);
      dequantise4(v[i].y, ex, c, d);
      E *at = dst + 2 * i * kGroupValues;
      if constexpr (sizeof(E) == 4) {
        reinterpret_cast<float4 *>(at)[0] = make_float4(f2_lo(a), f2_hi(a), f2_lo(b), f2_hi(b));
        reinterpret_cast<float4 *>(at)[1] = make_float4(f2_lo(c), f2_hi(c), f2_lo(d), f2_hi(d));
      } else {
        uint4 u;
        if constexpr (std::is_same<E, __half>::value) {
          const __half2 h[4] = {__floats2half2_rn(f2_lo(a), f2_hi(a)), __floats2half2_rn(f2_lo(b), f2_hi(b)),
                                __floats2half2_rn(f2_lo(c), f2_hi(c)), __floats2half2_rn(f2_lo(d), f2_hi(d))};
          memcpy(&u, h, sizeof(u));
        } else {
          u = make_uint4(pack_bf16x2(f2_lo(a), f2_hi(a)), pack_bf16x2(f2_lo(b), f2_hi(b)),
                         pack_bf16x2(f2_lo(c), f2_hi(c)), pack_bf16x2(f2_lo(d), f2_hi(d)));
        }
        *reinterpret_cast<uint4 *>(at) = u;
      }
    }
    return;
  }
  uint32_t q[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    q[i] = 0;
    if (i < n) {
      const Place at = place_of(t, item0 + i, true);
      const uint8_t *src = t.values + at.values;
      if constexpr (kVec) {
        if (4 * lane < at.left) q[i] = __ldg(reinterpret_cast<const uint32_t *>(src) + lane);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (lane + 32 * j < at.left) q[i] |= static_cast<uint32_t>(src[lane + 32 * j]) << (8 * j);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (i >= n) break;
    const Place at = place_of(t, item0 + i, true);
    uint64_t a, b;
    dequantise4(q[i], __shfl_sync(0xffffffffu, mine, i), a, b);
    store4<E, kVec>(static_cast<E *>(t.data) + at.data, lane, at.left, a, b);
  }
}

template <typename E>
cudaError_t launch_checkpoint_e(const Pack &p, uint32_t warps, bool vec, bool unpack, cudaStream_t stream) {
  const unsigned blocks = (warps + kWarps - 1) / kWarps;
  auto kernel = unpack ? (vec ? checkpoint_unpack_kernel<E, true> : checkpoint_unpack_kernel<E, false>)
                       : (vec ? checkpoint_pack_kernel<E, true> : checkpoint_pack_kernel<E, false>);
  kernel<<<blocks, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace rec
}  // namespace gdn
