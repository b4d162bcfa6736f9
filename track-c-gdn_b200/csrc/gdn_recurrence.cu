// gdn_recurrence.cu -- the channelwise gated linear recurrence for sm_100a:
// decode step, prefill over packed or dense sequences, and backward.
//
//   g_t = exp(-exp(A_log) softplus(a_t + dt_bias)),  beta_t = sigmoid(b_t)
//   h_t = g_t h_{t-1} + beta_t x_t,   out_t = h_t           (per channel, fp32)
//
// Prefill (gdn_recurrence_forward.cu) and backward (gdn_recurrence_backward.cu)
// cut the packed rows into chunks of 64, whatever the sequences' lengths, and the
// channels into tiles of 64 (128 where 8-bit copies are written), so that ragged
// batches load every SM alike.  A chunk maps the state before it to the state
// after it by one affine map per channel, h -> A h + H, with A the product of its
// gates; a chunk in which a sequence starts maps to a constant.  Backwards the
// same holds for R (see there) from the last row of a chunk to its first.
//
// Look-back: a chunk's map is published, its CTA fetches the maps of the chunks
// before it in its group of 8 and the state after the previous group, and applies
// them in order; the last chunk of a group publishes the state after it.  A serial
// chain thus has one link per 8 chunks.  Batches of several sequences are worked
// on in streams that run side by side (Stream in gdn_recurrence_tile.cuh); a
// chunk's predecessor is then done when its turn comes, and groups are of one.
// The order of all roundings is fixed by the sizes and cu_seqlens: results do not
// depend on timing.  Tiles are taken by ticket in the chain's order, so a CTA only
// ever waits for tiles that running CTAs have in hand, and every wait is bounded.
#include "gdn_recurrence_tile.cuh"

namespace gdn {
namespace rec {

// ---- decode --------------------------------------------------------------------
struct Decode {
  const void *x, *a, *b;
  int64_t x_stride, a_stride, b_stride;
  const float *A_log, *dt_bias;
  const float *state;
  const int32_t *slots;
  int64_t pool, B, D;
  int tokens;
  void *out;         // [B, tokens, D]
  float *new_state;  // rows of D
  float *inter;      // [B, tokens, D] or null
};

// A warp takes one request's 128 channels through its tokens, the state in
// registers: 8 bytes a channel and token and 8 for the state for 2-byte types,
// bound by HBM for large batches, by latency for small.  `out` may take the place
// of an input, so its loads are not of the read-only kind (1024 x 4 x 1024 bf16
// in a pool, not in L2: 13.5 us, 13.8 with those).
template <typename E, bool kVec>
__global__ void __launch_bounds__(kThreads) recurrence_decode_kernel(const __grid_constant__ Decode p) {
  const int lane = threadIdx.x & 31;
  const int nd = static_cast<int>((p.D + kTileCh - 1) / kTileCh);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= p.B * nd) return;
  const int64_t req = item / nd, c0 = item % nd * kTileCh;
  const int left = static_cast<int>(min(p.D - c0, int64_t{kTileCh}));
  const int64_t row = p.slots != nullptr ? p.slots[req] : req;
  if (p.slots != nullptr && (row < 0 || row >= p.pool)) {
    if (lane == 0) set_device_status(kDevStatusBadSlot);
    return;
  }
  float4 s = p.state != nullptr ? load_f32<kVec>(p.state + row * p.D + c0, lane, left)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
  uint64_t h[2] = {f2_pack(s.x, s.y), f2_pack(s.z, s.w)};
  const Params par = load_params<kVec>(p.A_log + c0, p.dt_bias + c0, lane, left);
#pragma unroll 2
  for (int i = 0; i < p.tokens; ++i) {
    const int64_t t = req * p.tokens + i;
    uint64_t x[2], a[2], b[2];
    load4<E, kVec, false>(static_cast<const E *>(p.x) + t * p.x_stride + c0, lane, left).pairs(x[0], x[1]);
    load4<E, kVec, false>(static_cast<const E *>(p.a) + t * p.a_stride + c0, lane, left).pairs(a[0], a[1]);
    load4<E, kVec, false>(static_cast<const E *>(p.b) + t * p.b_stride + c0, lane, left).pairs(b[0], b[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint64_t g, u;
      gate_pair(x[k], a[k], b[k], par.dt[k], par.c[k], g, u);
      h[k] = f2_fma(g, h[k], u);
    }
    store4<E, kVec>(static_cast<E *>(p.out) + t * p.D + c0, lane, left, h[0], h[1]);
    if (p.inter != nullptr)
      store_f32<kVec>(p.inter + t * p.D + c0, lane, left,
                      make_float4(f2_lo(h[0]), f2_hi(h[0]), f2_lo(h[1]), f2_hi(h[1])));
  }
  store_f32<kVec>(p.new_state + row * p.D + c0, lane, left,
                  make_float4(f2_lo(h[0]), f2_hi(h[0]), f2_lo(h[1]), f2_hi(h[1])));
}

// One token: all loads before the first use, nothing else in registers.  A warp
// to a request's 128 channels: two or four requests a warp, their loads all in
// flight at once, were no faster (4096 x 1024 bf16 in a pool, not in L2: 13.8 us,
// 4.9 TB/s; 14.0 and 14.4 us with two and four).
template <typename E, bool kVec>
__global__ void __launch_bounds__(kThreads) recurrence_decode_one_kernel(const __grid_constant__ Decode p) {
  const int lane = threadIdx.x & 31;
  const int nd = static_cast<int>((p.D + kTileCh - 1) / kTileCh);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= p.B * nd) return;
  const int64_t req = item / nd, c0 = item % nd * kTileCh;
  const int left = static_cast<int>(min(p.D - c0, int64_t{kTileCh}));
  const Raw<E> x = load4<E, kVec, false>(static_cast<const E *>(p.x) + req * p.x_stride + c0, lane, left);
  const Raw<E> a = load4<E, kVec, false>(static_cast<const E *>(p.a) + req * p.a_stride + c0, lane, left);
  const Raw<E> b = load4<E, kVec, false>(static_cast<const E *>(p.b) + req * p.b_stride + c0, lane, left);
  const Params par = load_params<kVec>(p.A_log + c0, p.dt_bias + c0, lane, left);
  const int64_t row = p.slots != nullptr ? p.slots[req] : req;
  if (p.slots != nullptr && (row < 0 || row >= p.pool)) {
    if (lane == 0) set_device_status(kDevStatusBadSlot);
    return;
  }
  const float4 s = p.state != nullptr ? load_f32<kVec>(p.state + row * p.D + c0, lane, left)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
  uint64_t xp[2], ap[2], bp[2], h[2] = {f2_pack(s.x, s.y), f2_pack(s.z, s.w)};
  x.pairs(xp[0], xp[1]);
  a.pairs(ap[0], ap[1]);
  b.pairs(bp[0], bp[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint64_t g, u;
    gate_pair(xp[k], ap[k], bp[k], par.dt[k], par.c[k], g, u);
    h[k] = f2_fma(g, h[k], u);
  }
  store4<E, kVec>(static_cast<E *>(p.out) + req * p.D + c0, lane, left, h[0], h[1]);
  store_f32<kVec>(p.new_state + row * p.D + c0, lane, left,
                  make_float4(f2_lo(h[0]), f2_hi(h[0]), f2_lo(h[1]), f2_hi(h[1])));
}

// ---- sizes and launches ----------------------------------------------------------
inline size_t saved_bytes(int64_t T, int64_t D) {  // the states before every 64th row
  return static_cast<size_t>(chunks_of(T) * tiles_of(D) * kTileCh * 4);
}

template <typename E>
cudaError_t launch_decode_e(const Decode &p, bool vec, cudaStream_t stream) {
  const int64_t blocks = (p.B * tiles_of(p.D) + kWarps - 1) / kWarps;
  auto kernel = p.tokens == 1 && p.inter == nullptr
                    ? (vec ? recurrence_decode_one_kernel<E, true> : recurrence_decode_one_kernel<E, false>)
                    : (vec ? recurrence_decode_kernel<E, true> : recurrence_decode_kernel<E, false>);
  kernel<<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace rec
}  // namespace gdn
