// gdn_recurrence.cu -- the channelwise gated linear recurrence for sm_100a:
// decode step, prefill over packed or dense sequences, and backward.
//
//   g_t = exp(-exp(A_log) softplus(a_t + dt_bias)),  beta_t = sigmoid(b_t)
//   h_t = g_t h_{t-1} + beta_t x_t,   out_t = h_t           (per channel, fp32)
//
// Prefill and backward cut the packed tokens into chunks of 64, whatever the
// sequences' lengths, and the channels into tiles of 128; a tile (chunk x 128
// channels) is one CTA's work, so ragged batches load every SM alike.  A
// chunk maps the state before it to the state after it by one affine map per
// channel, h -> A h + H, with A the product of its gates; a chunk in which a
// sequence starts maps to a constant.
//
// Look-back: the CTA of a chunk publishes its map, fetches the maps of the
// chunks before it in its group of 32 and the state after the previous group,
// and applies them in order; the last chunk of a group publishes the state
// after it.  A serial chain thus has one link per 32 chunks, and the order of
// all roundings is fixed: results do not depend on timing.  Tiles are taken
// by ticket in chunk order, so a CTA only ever waits for CTAs that already run.
#include "gdn_recurrence_tile.cuh"

namespace gdn {
namespace rec {

// The sequences that start or end in a chunk, by token of the chunk (-1: none).
struct ChunkSeqs {
  int start[kChunkTok], end[kChunkTok];
  int64_t lo, hi;
};

// Fills `cs` (all threads of the CTA; ends with a barrier).  on_empty(n) is
// called by whole warps for each sequence without tokens that lies in this
// chunk (the last chunk also has those behind the last token).
template <typename F>
__device__ __forceinline__ void find_sequences(const Seqs &s, ChunkSeqs &cs, int64_t base, bool last,
                                               int warp, int lane, F on_empty) {
  if (warp == 0) {
    const int64_t lo = first_at_or_after(s, base, lane);
    if (lane == 0) cs.lo = lo;
  } else if (warp == 1) {
    const int64_t hi = last ? s.N : first_at_or_after(s, base + kChunkTok, lane);
    if (lane == 0) cs.hi = hi;
  } else if (warp < 4) {
    int *t = warp == 2 ? cs.start : cs.end;
    t[lane] = t[lane + 32] = -1;
  }
  __syncthreads();
  const int64_t lo = cs.lo, hi = cs.hi;
  for (int64_t n0 = max(lo - 1, int64_t{0}) + warp * 32; n0 < hi; n0 += kThreads) {
    const int64_t n = n0 + lane;
    bool empty = false;
    if (n < hi) {
      const int64_t from = s.at(n), to = s.at(n + 1);
      empty = from == to && n >= lo;
      if (from < to) {
        if (from >= base && from < base + kChunkTok) cs.start[from - base] = static_cast<int>(n);
        if (to > base && to <= base + kChunkTok) cs.end[to - 1 - base] = static_cast<int>(n);
      }
    }
    unsigned m = __ballot_sync(0xffffffffu, empty);
    while (m) {
      on_empty(n0 + __ffs(m) - 1);
      m &= m - 1;
    }
  }
  __syncthreads();
}

// What the chain of chunks goes through: maps [position][tile][128], states
// after groups [group][tile][128].  Positions count in the chain's direction.
struct Chain {
  uint64_t *maps, *states;
};

struct Shared {
  float2 own[kWarps][kTileCh];       // maps of the warps' tokens
  float2 look[kWarps + 1][kTileCh];  // maps fetched by each warp; the group's state
  ChunkSeqs seqs;
  int ticket, broken;
};

// Joins maps of the CTA's warps [from, to) in steps of `dir`.
__device__ __forceinline__ Map4 identity() { return Map4{{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}}; }
__device__ __forceinline__ void advance(float (&h)[4], const float2 *row, int lane) {
  const Map4 m = get_map(row, lane);
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = apply(m.A[j], m.H[j], h[j]);
}

// Fetches what lies before position r of its group into sh.look (all warps;
// ends with a barrier) and returns the state that enters position r.
__device__ __forceinline__ void look_back(Shared &sh, const Chain &ch, int64_t r, int d, int nd, int warp,
                                          int lane, float (&h)[4]) {
  const int64_t first = r / kGroup * kGroup;
  const int count = static_cast<int>(r - first);
  if (warp * kLook < count) {
    Map4 m = identity();
#pragma unroll 1
    for (int k = 0; k < kLook; k += 2) {
      const int j = warp * kLook + k;
      if (j >= count) break;
      const uint64_t *src = ch.maps + ((first + j) * nd + d) * kTileCh;
      const bool two = j + 1 < count;
      uint64_t w0[4], w1[4];
      try_words(src, lane, w0);
      if (two) try_words(src + static_cast<int64_t>(nd) * kTileCh, lane, w1);
      if (!have_words(w0)) wait_words_slow(src, lane, w0, &sh.broken);
      compose(m, as_map(w0));
      if (two) {
        if (!have_words(w1)) wait_words_slow(src + static_cast<int64_t>(nd) * kTileCh, lane, w1, &sh.broken);
        compose(m, as_map(w1));
      }
    }
    put_map(sh.look[warp], lane, m);
  }
  if (warp == kWarps - 1 && first > 0) {
    const uint64_t *src = ch.states + ((first / kGroup - 1) * nd + d) * kTileCh;
    uint64_t w[4];
    try_words(src, lane, w);
    if (!have_words(w)) wait_words_slow(src, lane, w, &sh.broken);
    put_map(sh.look[kWarps], lane, as_map(w));
  }
  __syncthreads();
  if (first > 0) {
    const Map4 m = get_map(sh.look[kWarps], lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = m.H[j];
  }
  for (int i = 0; i * kLook < count; ++i) advance(h, sh.look[i], lane);
}

// Zeros in rows [from, to) of the tile's channels of p [T, D].
template <typename E, bool kVec>
__device__ __forceinline__ void zero_rows(void *p, int64_t from, int64_t to, int64_t D, int64_t c0, int warp,
                                          int lane, int left) {
  for (int64_t t = from + warp; t < to; t += kWarps)
    store4<E, kVec>(static_cast<E *>(p) + t * D + c0, lane, left, 0, 0);
}

// ---- backward ------------------------------------------------------------------
//   dh_t = d_out_t + R_t,  R_{t-1} = g_t dh_t  (R_t = d_final at a last token)
//   dx = beta dh,  db = x dh beta (1 - beta),  dlg = g h_{t-1} dh
//   da = -exp(A_log) dlg sigmoid(z),  ddt_bias = sum da,  dA_log = sum dlg lg
//   d_state = g dh of a first token
// One pass from the last chunk to the first: the states before the tokens come
// from the state saved at the chunk's start, R runs through the chain.
struct Backward {
  const void *x, *a, *b, *d_out;
  int64_t x_stride, a_stride, b_stride, do_stride;
  const uint8_t *packed;  // 8-bit x, a, b instead (kPacked)
  const float *A_log, *dt_bias, *state, *d_final;
  const float *carries;
  Seqs s;
  int64_t D;
  void *dx, *da, *db;  // [T, D]
  float *d_state;      // [N, D], or null
  float2 *partials;    // [chunk][tile][128] (sum dlg lg, sum da), lane order
  int zero_behind;     // write zeros to dx, da, db behind the last sequence
  Header *hdr;
  Chain chain;
};

template <typename E, bool kVec, bool kPacked>
struct Inputs {
  __device__ static __forceinline__ void load(const Backward &p, int64_t t, int64_t c0, int d, int nd, int lane,
                                              int left, uint64_t (&x)[2], uint64_t (&a)[2], uint64_t (&b)[2]) {
    if constexpr (kPacked) {
      uint64_t *v[3] = {x, a, b};
#pragma unroll
      for (int w = 0; w < 3; ++w) {
        const uint8_t *src = p.packed + (w * p.s.T + t) * p.D + c0;
        uint32_t q = 0;
        if constexpr (kVec) {
          if (4 * lane < left) q = __ldg(reinterpret_cast<const uint32_t *>(src) + lane);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (lane + 32 * j < left) q |= static_cast<uint32_t>(src[lane + 32 * j]) << (8 * j);
        }
        const uint32_t ex = __ldg(p.packed + 3 * p.s.T * p.D + (w * p.s.T + t) * nd + d);
        dequantise4(q, ex, v[w][0], v[w][1]);
      }
    } else {
      load4<E, kVec>(static_cast<const E *>(p.x) + t * p.x_stride + c0, lane, left).pairs(x[0], x[1]);
      load4<E, kVec>(static_cast<const E *>(p.a) + t * p.a_stride + c0, lane, left).pairs(a[0], a[1]);
      load4<E, kVec>(static_cast<const E *>(p.b) + t * p.b_stride + c0, lane, left).pairs(b[0], b[1]);
    }
  }
};

template <typename E, bool kVec, bool kPacked>
__global__ void __launch_bounds__(kThreads, 2)
recurrence_backward_kernel(const __grid_constant__ Backward p) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nd = static_cast<int>((p.D + kTileCh - 1) / kTileCh);
  if (tid == 0) {
    sh.broken = 0;
    sh.ticket = p.hdr->bad ? -1 : static_cast<int>(atomicAdd(&p.hdr->stream[0].ticket, 1u));
  }
  __syncthreads();
  if (sh.ticket < 0) return;
  const int64_t total = p.s.total();
  const int64_t last = total > 0 ? (total - 1) / kChunkTok : 0;
  const int64_t r = sh.ticket / nd, chunk = last - r;  // position in the chain, from the end
  const int d = sh.ticket % nd;
  const int64_t c0 = static_cast<int64_t>(d) * kTileCh;
  const int left = static_cast<int>(min(p.D - c0, int64_t{kTileCh}));
  if (p.zero_behind) {  // position r has chunk r's rows to zero
    const int64_t from = max(r * kChunkTok, total), to = min((r + 1) * kChunkTok, p.s.T);
    zero_rows<E, kVec>(p.dx, from, to, p.D, c0, warp, lane, left);
    zero_rows<E, kVec>(p.da, from, to, p.D, c0, warp, lane, left);
    zero_rows<E, kVec>(p.db, from, to, p.D, c0, warp, lane, left);
  }
  if (chunk < 0) return;
  const Params par = load_params<kVec>(p.A_log + c0, p.dt_bias + c0, lane, left);
  const int64_t base = chunk * kChunkTok, t0 = base + warp * kTok;
  const int valid = static_cast<int>(max(int64_t{0}, min(int64_t{kTok}, total - t0)));
  const float4 zero4 = make_float4(0.f, 0.f, 0.f, 0.f);

  uint64_t g[kTok][2], u[kTok][2], o[kTok][2];
#pragma unroll
  for (int i = 0; i < kTok; ++i) {
    g[i][0] = g[i][1] = f2_dup(1.f);
    u[i][0] = u[i][1] = o[i][0] = o[i][1] = 0;
    if (i < valid) {
      uint64_t x[2], a[2], b[2];
      Inputs<E, kVec, kPacked>::load(p, t0 + i, c0, d, nd, lane, left, x, a, b);
      load4<E, kVec>(static_cast<const E *>(p.d_out) + (t0 + i) * p.do_stride + c0, lane, left).pairs(o[i][0], o[i][1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) gate_pair(x[k], a[k], b[k], par.dt[k], par.c[k], g[i][k], u[i][k]);
    }
  }
  find_sequences(p.s, sh.seqs, base, chunk == last, warp, lane, [&](int64_t n) {
    if (p.d_state == nullptr) return;  // an empty sequence's final state is its initial state
    store_f32<kVec>(p.d_state + n * p.D + c0, lane, left,
                    p.d_final != nullptr ? load_f32<kVec>(p.d_final + n * p.D + c0, lane, left) : zero4);
  });
  const unsigned starts = __ballot_sync(0xffffffffu, lane < kTok && sh.seqs.start[warp * kTok + (lane & 7)] >= 0);
  const unsigned ends = __ballot_sync(0xffffffffu, lane < kTok && sh.seqs.end[warp * kTok + (lane & 7)] >= 0);
  const bool enters = sh.seqs.end[kChunkTok - 1] < 0 && chunk < last;

  // maps of the warp's tokens: of the state forwards, of R backwards
  {
    uint64_t A2[2] = {f2_dup(1.f), f2_dup(1.f)}, H2[2] = {0, 0}, B2[2] = {f2_dup(1.f), f2_dup(1.f)}, R2[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      if ((starts >> i) & 1) {
        const float4 v = p.state != nullptr
                             ? load_f32<kVec>(p.state + sh.seqs.start[warp * kTok + i] * p.D + c0, lane, left)
                             : zero4;
        H2[0] = f2_fma(g[i][0], f2_pack(v.x, v.y), u[i][0]);
        H2[1] = f2_fma(g[i][1], f2_pack(v.z, v.w), u[i][1]);
        A2[0] = A2[1] = f2_dup(-1.f);
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) A2[k] = f2_mul(A2[k], g[i][k]), H2[k] = f2_fma(g[i][k], H2[k], u[i][k]);
      }
    }
#pragma unroll
    for (int i = kTok - 1; i >= 0; --i) {
      if ((ends >> i) & 1) {
        const float4 v = p.d_final != nullptr
                             ? load_f32<kVec>(p.d_final + sh.seqs.end[warp * kTok + i] * p.D + c0, lane, left)
                             : zero4;
        R2[0] = f2_pack(v.x, v.y);
        R2[1] = f2_pack(v.z, v.w);
        B2[0] = B2[1] = f2_dup(-1.f);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) B2[k] = f2_mul(B2[k], g[i][k]), R2[k] = f2_mul(g[i][k], f2_add(o[i][k], R2[k]));
    }
    put_map(sh.own[warp], lane,
            Map4{{f2_lo(A2[0]), f2_hi(A2[0]), f2_lo(A2[1]), f2_hi(A2[1])},
                 {f2_lo(H2[0]), f2_hi(H2[0]), f2_lo(H2[1]), f2_hi(H2[1])}});
    __syncthreads();
    // the state before the warp's first token, then g h_{t-1} of each token in u's place
    const float4 c = load_f32<kVec>(p.carries + (chunk * nd + d) * kTileCh, lane, kTileCh);
    float h[4] = {c.x, c.y, c.z, c.w};
    for (int i = 0; i < warp; ++i) advance(h, sh.own[i], lane);
    uint64_t s2[2] = {f2_pack(h[0], h[1]), f2_pack(h[2], h[3])};
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      if ((starts >> i) & 1) {
        const float4 v = p.state != nullptr
                             ? load_f32<kVec>(p.state + sh.seqs.start[warp * kTok + i] * p.D + c0, lane, left)
                             : zero4;
        s2[0] = f2_pack(v.x, v.y);
        s2[1] = f2_pack(v.z, v.w);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint64_t gh = f2_mul(g[i][k], s2[k]);
        s2[k] = f2_fma(g[i][k], s2[k], u[i][k]);
        u[i][k] = gh;
      }
    }
    __syncthreads();
    put_map(sh.own[warp], lane,
            Map4{{f2_lo(B2[0]), f2_hi(B2[0]), f2_lo(B2[1]), f2_hi(B2[1])},
                 {f2_lo(R2[0]), f2_hi(R2[0]), f2_lo(R2[1]), f2_hi(R2[1])}});
    __syncthreads();
  }

  float R[4] = {0.f, 0.f, 0.f, 0.f};
  const bool group_end = r % kGroup == kGroup - 1;
  if (warp == kWarps - 1 && chunk > 0 && !group_end) {
    Map4 m = get_map(sh.own[kWarps - 1], lane);
    for (int i = kWarps - 2; i >= 0; --i) compose(m, get_map(sh.own[i], lane));
    put_words(p.chain.maps + (r * nd + d) * kTileCh, lane, m.A, m.H);
  }
  if (enters) look_back(sh, p.chain, r, d, nd, warp, lane, R);
  if (warp == 0 && chunk > 0 && group_end) {
    float Rg[4] = {R[0], R[1], R[2], R[3]};
    for (int i = kWarps - 1; i >= 0; --i) advance(Rg, sh.own[i], lane);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    put_words(p.chain.states + (r / kGroup * nd + d) * kTileCh, lane, zero, Rg);
  }
  for (int i = kWarps - 1; i > warp; --i) advance(R, sh.own[i], lane);

  uint64_t R2[2] = {f2_pack(R[0], R[1]), f2_pack(R[2], R[3])};
  uint64_t sum_lg[2] = {0, 0}, sum_da[2] = {0, 0};
  constexpr float kLn2 = 0.6931471805599453f;
#pragma unroll
  for (int i = kTok - 1; i >= 0; --i) {
    if (i < valid) {
      uint64_t x[2], a[2], b[2], dx[2], da[2], db[2];
      Inputs<E, kVec, kPacked>::load(p, t0 + i, c0, d, nd, lane, left, x, a, b);
      if ((ends >> i) & 1) {
        const float4 v = p.d_final != nullptr
                             ? load_f32<kVec>(p.d_final + sh.seqs.end[warp * kTok + i] * p.D + c0, lane, left)
                             : zero4;
        R2[0] = f2_pack(v.x, v.y);
        R2[1] = f2_pack(v.z, v.w);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint64_t dh = f2_add(o[i][k], R2[k]);
        R2[k] = f2_mul(g[i][k], dh);
        // beta and beta (1 - beta) from e = exp(-|b|): r = 1 / (1 + e), e r
        const uint64_t eb = ex2_neg_abs(f2_mul(b[k], f2_dup(kLog2e))), db1 = f2_add(eb, f2_dup(1.f));
        const uint64_t rb = f2_pack(rcp(f2_lo(db1)), rcp(f2_hi(db1))), erb = f2_mul(eb, rb);
        const uint64_t beta = f2_pack(f2_lo(b[k]) >= 0.f ? f2_lo(rb) : f2_lo(erb),
                                      f2_hi(b[k]) >= 0.f ? f2_hi(rb) : f2_hi(erb));
        dx[k] = f2_mul(beta, dh);
        db[k] = f2_mul(f2_mul(x[k], dh), f2_mul(rb, erb));
        const uint64_t z = f2_fma(a[k], f2_dup(kLog2e), par.dt[k]), e = ex2_neg_abs(z), d1 = f2_add(e, f2_dup(1.f));
        const uint64_t rz = f2_pack(rcp(f2_lo(d1)), rcp(f2_hi(d1))), erz = f2_mul(e, rz);
        const uint64_t sig = f2_pack(f2_lo(z) >= 0.f ? f2_lo(rz) : f2_lo(erz),
                                     f2_hi(z) >= 0.f ? f2_hi(rz) : f2_hi(erz));
        const uint64_t cd = f2_mul(par.c[k], f2_mul(u[i][k], dh));  // -exp(A_log) dlg
        da[k] = f2_mul(cd, sig);
        sum_da[k] = f2_add(sum_da[k], da[k]);
        sum_lg[k] = f2_fma(cd, softplus2(z, e), sum_lg[k]);  // dlg lg log2(e)
      }
      const int64_t at = (t0 + i) * p.D + c0;
      store4<E, kVec>(static_cast<E *>(p.dx) + at, lane, left, dx[0], dx[1]);
      store4<E, kVec>(static_cast<E *>(p.da) + at, lane, left, da[0], da[1]);
      store4<E, kVec>(static_cast<E *>(p.db) + at, lane, left, db[0], db[1]);
      if (((starts >> i) & 1) && p.d_state != nullptr)
        store_f32<kVec>(p.d_state + sh.seqs.start[warp * kTok + i] * p.D + c0, lane, left,
                        make_float4(f2_lo(R2[0]), f2_hi(R2[0]), f2_lo(R2[1]), f2_hi(R2[1])));
    }
  }
  sum_lg[0] = f2_mul(sum_lg[0], f2_dup(kLn2));
  sum_lg[1] = f2_mul(sum_lg[1], f2_dup(kLn2));
  // the chunk's part of the parameters' gradients, over the warps in order
  __syncthreads();
  put_map(sh.own[warp], lane,
          Map4{{f2_lo(sum_lg[0]), f2_hi(sum_lg[0]), f2_lo(sum_lg[1]), f2_hi(sum_lg[1])},
               {f2_lo(sum_da[0]), f2_hi(sum_da[0]), f2_lo(sum_da[1]), f2_hi(sum_da[1])}});
  __syncthreads();
  if (tid < kTileCh) {
    float2 v = sh.own[0][tid];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v.x += sh.own[i][tid].x, v.y += sh.own[i][tid].y;
    p.partials[(chunk * nd + d) * kTileCh + tid] = v;
  }
}

// Sums the chunks' parts in a fixed order: 32 threads of a channel take every
// 32nd chunk, then their sums are added.  dlg lg needs no factor; see above.
template <bool kVec>
__global__ void __launch_bounds__(1024)
recurrence_params_kernel(const float2 *partials, const Header *hdr, const Seqs s, int64_t D, int nd,
                         float *dA_log, float *ddt_bias) {
  __shared__ float2 part[32][33];
  if (hdr->bad) return;
  const int64_t total = s.total();
  const int64_t chunks = total > 0 ? (total - 1) / kChunkTok + 1 : 0;
  const int d = blockIdx.x / 4, slot = (blockIdx.x % 4) * 32 + threadIdx.x;
  float2 v = make_float2(0.f, 0.f);
#pragma unroll 8
  for (int64_t c = threadIdx.y; c < chunks; c += 32) {
    const float2 q = partials[(c * nd + d) * kTileCh + slot];
    v.x += q.x;
    v.y += q.y;
  }
  part[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0) {
    for (int i = 1; i < 32; ++i) v.x += part[i][threadIdx.x].x, v.y += part[i][threadIdx.x].y;
    const int64_t c = static_cast<int64_t>(d) * kTileCh + lane_channel<kVec>(slot >> 2, slot & 3);
    if (c < D) {
      dA_log[c] = v.x;
      ddt_bias[c] = v.y;
    }
  }
}

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
// registers: 16 bytes a channel and token for 2-byte types (state in and out
// and four vectors), bound by HBM for large batches, by latency for small.
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
    load4<E, kVec>(static_cast<const E *>(p.x) + t * p.x_stride + c0, lane, left).pairs(x[0], x[1]);
    load4<E, kVec>(static_cast<const E *>(p.a) + t * p.a_stride + c0, lane, left).pairs(a[0], a[1]);
    load4<E, kVec>(static_cast<const E *>(p.b) + t * p.b_stride + c0, lane, left).pairs(b[0], b[1]);
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

// ---- sizes and launches ----------------------------------------------------------
inline size_t saved_bytes(int64_t T, int64_t D) {  // carries
  return static_cast<size_t>(chunks_of(T) * tiles_of(D) * kTileCh * 4);
}

template <typename E, bool kVec, bool kPacked>
cudaError_t launch_backward_t(Backward p, void *workspace, float *dA_log, float *ddt_bias, cudaStream_t stream) {
  const int64_t nd = tiles_of(p.D);
  p.hdr = static_cast<Header *>(workspace);
  const Places w = places(workspace, p.s.T, p.D);
  p.chain.maps = w.words;
  p.chain.states = p.chain.maps + chunks_of(p.s.T) * nd * kTileCh;
  const Prepared q{p.A_log, p.dt_bias, w.dt, w.c, p.D, nullptr, chunks_of(p.s.T), kRows, 1};
  const int64_t words = (chunks_of(p.s.T) + (chunks_of(p.s.T) + kGroupLen - 1) / kGroupLen) * nd * kTileCh;
  if (cudaError_t e = launch_init(p.hdr, w.words, words, p.s, q, stream)) return e;
  recurrence_backward_kernel<E, kVec, kPacked>
      <<<static_cast<unsigned>(chunks_of(p.s.T) * nd), kThreads, 0, stream>>>(p);
  if (cudaError_t e = cudaGetLastError()) return e;
  recurrence_params_kernel<kVec><<<static_cast<unsigned>(nd * 4), dim3(32, 32), 0, stream>>>(
      p.partials, p.hdr, p.s, p.D, static_cast<int>(nd), dA_log, ddt_bias);
  return cudaGetLastError();
}

template <typename E>
cudaError_t launch_backward_e(const Backward &p, bool vec, void *workspace, float *dA_log, float *ddt_bias,
                              cudaStream_t stream) {
  if (p.packed != nullptr)
    return vec ? launch_backward_t<E, true, true>(p, workspace, dA_log, ddt_bias, stream)
               : launch_backward_t<E, false, true>(p, workspace, dA_log, ddt_bias, stream);
  return vec ? launch_backward_t<E, true, false>(p, workspace, dA_log, ddt_bias, stream)
             : launch_backward_t<E, false, false>(p, workspace, dA_log, ddt_bias, stream);
}

template <typename E>
cudaError_t launch_decode_e(const Decode &p, bool vec, cudaStream_t stream) {
  const int64_t blocks = (p.B * tiles_of(p.D) + kWarps - 1) / kWarps;
  auto kernel = vec ? recurrence_decode_kernel<E, true> : recurrence_decode_kernel<E, false>;
  kernel<<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace rec
}  // namespace gdn
