// gdn_checkpoint.cu -- activations to int8 groups and back (format in
// gdn_recurrence.cuh: 128 values of a row share one power of two).
//
// A warp takes kPackRows groups at once, loads them all before it works on the
// first, finds each group's largest magnitude with one warp reduction on the
// fp32 bits, and writes a byte per value and a byte per group.  Bound by HBM:
// 3 bytes a value each way for 2-byte types.
#include "gdn_recurrence.cuh"

namespace gdn {
namespace rec {

constexpr int kPackTensors = 4;  // tensors of one launch
constexpr int kPackRows = 4;

struct PackTensor {
  const void *data;  // pack: the input; unpack: unused
  void *out;         // unpack: the output [rows, cols]
  uint8_t *values;   // [rows, cols] int8
  uint8_t *scales;   // [rows, groups]
  int64_t inner, outer_stride, inner_stride;  // row r lies at r / inner, r % inner
  int64_t cols, groups;
  int64_t first;     // number of the tensor's first group in the launch
};
struct Pack {
  PackTensor t[kPackTensors];
  int count;
  int64_t items;
};

// The tensor that group `item` belongs to (an index, so that the launch
// argument is not copied).
__device__ __forceinline__ int tensor_of(const Pack &p, int64_t item) {
  int k = 0;
#pragma unroll
  for (int i = 1; i < kPackTensors; ++i) k = i < p.count && item >= p.t[i].first ? i : k;
  return k;
}

template <typename E, bool kVec>
__global__ void __launch_bounds__(kThreads) checkpoint_pack_kernel(const __grid_constant__ Pack p) {
  const int lane = threadIdx.x & 31;
  const int64_t item0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kPackRows;
  Raw<E> raw[kPackRows];
  int left[kPackRows];
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    raw[i] = {};
    left[i] = 0;
    if (item0 + i < p.items) {
      const PackTensor &t = p.t[tensor_of(p, item0 + i)];
      const int64_t n = item0 + i - t.first, row = n / t.groups, c0 = n % t.groups * kGroupValues;
      left[i] = static_cast<int>(min(t.cols - c0, int64_t{kGroupValues}));
      raw[i] = load4<E, kVec>(static_cast<const E *>(t.data) + row / t.inner * t.outer_stride +
                                  row % t.inner * t.inner_stride + c0, lane, left[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    if (item0 + i >= p.items) break;
    const PackTensor &t = p.t[tensor_of(p, item0 + i)];
    const int64_t n = item0 + i - t.first, row = n / t.groups, c0 = n % t.groups * kGroupValues;
    uint64_t a, b;
    raw[i].pairs(a, b);
    const uint32_t ex = group_exponent(__reduce_max_sync(0xffffffffu, abs_max_bits(a, b)), exp_cap<E>());
    const uint32_t q = quantise4(a, b, ex, exp_cap<E>());
    uint8_t *dst = t.values + row * t.cols + c0;
    if constexpr (kVec) {
      if (4 * lane < left[i]) reinterpret_cast<uint32_t *>(dst)[lane] = q;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lane + 32 * j < left[i]) dst[lane + 32 * j] = static_cast<uint8_t>(q >> (8 * j));
    }
    if (lane == 0) t.scales[n] = static_cast<uint8_t>(ex);
  }
}

template <typename E, bool kVec>
__global__ void __launch_bounds__(kThreads) checkpoint_unpack_kernel(const __grid_constant__ Pack p) {
  const int lane = threadIdx.x & 31;
  const int64_t item0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kPackRows;
  uint32_t q[kPackRows], ex[kPackRows];
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    q[i] = ex[i] = 0;
    if (item0 + i < p.items) {
      const PackTensor &t = p.t[tensor_of(p, item0 + i)];
      const int64_t n = item0 + i - t.first, row = n / t.groups, c0 = n % t.groups * kGroupValues;
      const int left = static_cast<int>(min(t.cols - c0, int64_t{kGroupValues}));
      const uint8_t *src = t.values + row * t.cols + c0;
      ex[i] = __ldg(t.scales + n);
      if constexpr (kVec) {
        if (4 * lane < left) q[i] = __ldg(reinterpret_cast<const uint32_t *>(src) + lane);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (lane + 32 * j < left) q[i] |= static_cast<uint32_t>(src[lane + 32 * j]) << (8 * j);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    if (item0 + i >= p.items) break;
    const PackTensor &t = p.t[tensor_of(p, item0 + i)];
    const int64_t n = item0 + i - t.first, row = n / t.groups, c0 = n % t.groups * kGroupValues;
    uint64_t a, b;
    dequantise4(q[i], ex[i], a, b);
    store4<E, kVec>(static_cast<E *>(t.out) + row * t.cols + c0, lane,
                    static_cast<int>(min(t.cols - c0, int64_t{kGroupValues})), a, b);
  }
}

template <typename E>
cudaError_t launch_checkpoint_e(const Pack &p, bool vec, bool unpack, cudaStream_t stream) {
  const int64_t per_block = kWarps * kPackRows;
  const unsigned blocks = static_cast<unsigned>((p.items + per_block - 1) / per_block);
  auto kernel = unpack ? (vec ? checkpoint_unpack_kernel<E, true> : checkpoint_unpack_kernel<E, false>)
                       : (vec ? checkpoint_pack_kernel<E, true> : checkpoint_pack_kernel<E, false>);
  kernel<<<blocks, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace rec
}  // namespace gdn
