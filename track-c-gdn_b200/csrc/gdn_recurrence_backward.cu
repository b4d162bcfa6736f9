// gdn_recurrence_backward.cu -- gradients of the channelwise gated linear
// recurrence (mathematics and look-back: gdn_recurrence.cu).
//
//   dh_t = d_out_t + R_t,  R_{t-1} = g_t dh_t  (R_t = d_final at a last token)
//   dx = beta dh,  db = x dh beta (1 - beta),  dlg = g h_{t-1} dh
//   da = -exp(A_log) dlg sigmoid(z),  ddt_bias = sum da,  dA_log = sum dlg lg
//   d_state = g dh of a first token
//
// One pass over the tiles from the last chunk to the first, with the roles of
// the forward.  The state that enters a chunk was saved; R goes through the
// chain.  Consumers, first pass: the slot's map of the state (P, y) and of R
// (P, Q with Q = sum of P_i d_out_i: one ascending sweep gives both); softplus
// and beta stay in shared memory.  Second pass, when the chain warp has what
// enters: half a slot (4 rows) at a time, first upwards for the states, then
// downwards for the gradients.
//
// What bounds it: instructions (66 of a warp for 32 values, 2.2 a cycle of 4).
// 8 x 4096 x 2048 bf16 takes 216 us (4.3 TB/s; 144 us at the rate of a copy),
// from 8-bit x, a, b 252 us: converting bytes costs more than they save to read.
#include "gdn_recurrence_tile.cuh"

namespace gdn {
namespace rec {

template <typename E, Fetch kFetch, bool kPacked>
struct BwdShape {
  static constexpr int kThreads = 32 * (kSlots + 2);
  static constexpr int kPitch = row_pitch<static_cast<int>(sizeof(E))>(kFetch);  // of d_out; of x, a, b
  static constexpr int kInPitch = kPacked ? row_pitch<1>(kFetch) : kPitch;
  static constexpr int kPlane = kRows * kPitch, kInPlane = kRows * kInPitch;
  static constexpr int kStage = kPlane + 3 * kInPlane;
  static constexpr int kStages = 2;
  static constexpr int kCtas = kStage > 49152 ? 1 : 2;
};

struct Backward {
  CUtensorMap tx, ta, tb, to;  // kTmaTile
  const void *x, *a, *b, *d_out;
  int64_t x_stride, a_stride, b_stride, do_stride;
  const uint8_t *packed;  // 8-bit x, a, b instead (kPacked)
  const float *A_log, *dt_bias, *state, *d_final;
  const float *carries;
  Seqs s;
  int64_t D;
  void *dx, *da, *db;  // [T, D]
  float *d_state;      // [N, D], or null
  float2 *partials;    // [chunk][D up to 128s] (sum dlg lg, sum da)
  int zero_behind;     // write zeros to dx, da, db behind the last sequence
  Header *hdr;
  uint64_t *maps, *states;
  const float *dt, *c;
  const int *first;
};

template <typename Shape, bool kPacked>
struct BwdShared {
  // A slot's P and y, and its Q.  The chain warp replaces P, y by the state and
  // the R that enter.
  float4 own[kSlots][32];
  float2 rev[kSlots][32];
  // what the first pass leaves to the second: softplus(z) log2(e) and beta
  ulonglong2 kept[kSlots][kTokW][32];
  float params[Shape::kStages][2][64];
  uint8_t scales[kPacked ? Shape::kStages : 1][3][kRows];
  Table<kRows> tables[Shape::kStages];
  Tile tiles[Shape::kStages];
  uint64_t full[Shape::kStages], ready[Shape::kStages], empty[Shape::kStages];
  uint64_t mapped[Shape::kStages], taken[Shape::kStages];
  int broken;
};

template <typename E, Fetch kFetch, bool kPacked>
__global__ void __launch_bounds__(BwdShape<E, kFetch, kPacked>::kThreads, BwdShape<E, kFetch, kPacked>::kCtas)
recurrence_backward_kernel(const __grid_constant__ Backward p) {
  using S = BwdShape<E, kFetch, kPacked>;
  constexpr bool kVec = kFetch == kTmaTile;
  constexpr int kElement = sizeof(E), kInElement = kPacked ? 1 : kElement;
  constexpr int kStages = S::kStages;
  extern __shared__ __align__(1024) unsigned char smem[];
  BwdShared<S, kPacked> &sh = *reinterpret_cast<BwdShared<S, kPacked> *>(smem + kStages * S::kStage);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nt = static_cast<int>((p.D + 63) / 64);
  const int64_t groups128 = (p.D + 127) / 128;
  if (p.hdr->bad) return;
  if (tid == 0) {
    sh.broken = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&sh.full[i]), fetch_arrivals(kFetch));
      mbar_init(smem_u32(&sh.mapped[i]), kSlots);
      mbar_init(smem_u32(&sh.taken[i]), 1);
      mbar_init(smem_u32(&sh.ready[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), kSlots);
    }
    mbar_init_fence();
  }
  __syncthreads();
  const int64_t total = p.s.total();
  const int64_t last = total > 0 ? (total - 1) / kRows : 0;
  const int group_len = p.hdr->group;  // 1 or kGroupLen
  uint64_t *const states = group_len == 1 ? p.maps : p.states;

  auto input = [&](int w) -> const void * {
    if (kPacked) return p.packed + w * p.s.T * p.D;
    return w == 0 ? p.x : w == 1 ? p.a : p.b;
  };
  auto input_stride = [&](int w) { return kPacked ? p.D : w == 0 ? p.x_stride : w == 1 ? p.a_stride : p.b_stride; };

  if (warp == kSlots) {
    // ---- producer ----
    int left_streams = p.hdr->streams;
    int stream = blockIdx.x % left_streams;
    Stream st = p.hdr->stream[stream];
    uint32_t ticket = 0;
    if (lane == 0) ticket = atomicAdd(&p.hdr->stream[stream].ticket, 1u);
    int k = 0;
    // a tile's sums for the parameters' gradients, over the slots in order
    auto finish = [&](int i) {
      const int s = i % kStages;
      if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.empty[s]), (i / kStages) & 1, &sh.broken))) return false;
      const Table<kRows> &t = sh.tables[s];
      if (!t.only_map) {
        const unsigned char *sums = smem + s * S::kStage + lane * 16;
        float4 v = *reinterpret_cast<const float4 *>(sums);
#pragma unroll
        for (int j = 1; j < kSlots; ++j) {
          const float4 w = *reinterpret_cast<const float4 *>(sums + j * (S::kPlane / kSlots));
          v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
        float2 *dst = p.partials + t.chunk * groups128 * 128 + t.d * 64;
        if constexpr (kVec) {
          reinterpret_cast<float4 *>(dst)[lane] = make_float4(v.x, v.z, v.y, v.w);
        } else {
          dst[lane] = make_float2(v.x, v.z);
          dst[lane + 32] = make_float2(v.y, v.w);
        }
      }
      __syncwarp();
      return true;
    };
    while (true) {
      int64_t chunk = -1;
      int d = 0;
      bool only_map = false;
      const int64_t t0 = __shfl_sync(0xffffffffu, ticket, 0);
      if (left_streams > 0) {
        if (t0 < (st.to - st.from + st.only_map) * nt) {
          if (lane == 0) ticket = atomicAdd(&p.hdr->stream[stream].ticket, 1u);  // the next one, early
          chunk = st.to - 1 + st.only_map - t0 / nt;
          only_map = chunk == st.to;
          d = static_cast<int>(t0 % nt);
        } else if (--left_streams > 0) {
          stream = stream + 1 == p.hdr->streams ? 0 : stream + 1;
          st = p.hdr->stream[stream];
          if (lane == 0) ticket = atomicAdd(&p.hdr->stream[stream].ticket, 1u);
          continue;
        }
      }
      const int64_t c0 = static_cast<int64_t>(d) * 64, base = chunk * kRows;
      GDN_DCHECK(chunk < 0 || (d >= 0 && d < nt && base < max(p.s.T, int64_t{1})));
      const int left = static_cast<int>(min(p.D - c0, int64_t{64}));
      if (chunk >= 0 && p.zero_behind && !only_map) {
        for (int64_t t = max(base, total); t < min(base + kRows, p.s.T); ++t) {
          store2<E, kVec>(static_cast<E *>(p.dx) + t * p.D + c0, lane, left, 0);
          store2<E, kVec>(static_cast<E *>(p.da) + t * p.D + c0, lane, left, 0);
          store2<E, kVec>(static_cast<E *>(p.db) + t * p.D + c0, lane, left, 0);
        }
      }
      if (chunk > last) continue;
      const int s = k % kStages;
      if (k >= kStages && !finish(k - kStages)) break;
      Table<kRows> &t = sh.tables[s];
      const uint32_t full = smem_u32(&sh.full[s]);
      if (chunk < 0) {
        if (lane == 0) {
          t.chunk = -1;
          sh.tiles[s].d = -1;
          mbar_arrive(full);
        }
        if (kFetch == kRowCopies) mbar_arrive(full);
        for (int i = max(k - kStages + 1, 0); i < k; ++i)
          if (!finish(i)) break;
        break;
      }
      if (lane == 0) {
        mbar_expect_tx(full, 2 * 64 * 4 + (kVec ? S::kStage : 0));
        bulk_load(smem_u32(sh.params[s][0]), p.dt + c0, 64 * 4, full);
        bulk_load(smem_u32(sh.params[s][1]), p.c + c0, 64 * 4, full);
        if constexpr (kFetch == kTmaTile) {
          const uint32_t dst = smem_u32(smem + s * S::kStage);
          const int x = static_cast<int>(c0), y = static_cast<int>(base);
          tma_load_2d(dst, &p.to, x, y, full);
          tma_load_2d(dst + S::kPlane, &p.tx, x, y, full);
          tma_load_2d(dst + S::kPlane + S::kInPlane, &p.ta, x, y, full);
          tma_load_2d(dst + S::kPlane + 2 * S::kInPlane, &p.tb, x, y, full);
        }
      }
      if constexpr (kFetch == kRowCopies) {
        const int rows = static_cast<int>(min(total - base, int64_t{kRows}));
        const uint32_t dst = smem_u32(smem + s * S::kStage);
        copy_rows<kElement>(dst, p.d_out, p.do_stride, base, rows, c0, left, lane);
#pragma unroll
        for (int w = 0; w < 3; ++w)
          copy_rows<kInElement>(dst + S::kPlane + w * S::kInPlane, input(w), input_stride(w), base, rows, c0, left,
                                lane);
        arrive_after_copies(full);
      }
      if constexpr (kPacked) {
#pragma unroll
        for (int w = 0; w < 3; ++w)
#pragma unroll
          for (int i = 0; i < kRows; i += 32)
            sh.scales[s][w][i + lane] =
                base + i + lane < p.s.T
                    ? __ldg(p.packed + 3 * p.s.T * p.D + (w * p.s.T + base + i + lane) * groups128 + d / 2)
                    : 0;
      }
      const bool inside = fill_table<kRows>(p.s, t, base, chunk == last, lane, p.first, [&](int64_t n) {
        if (p.d_state == nullptr || only_map) return;  // an empty sequence's final state is its initial state
        store2_f32<kVec>(p.d_state + n * p.D + c0, lane, left,
                         p.d_final != nullptr ? load2_f32<kVec>(p.d_final + n * p.D + c0, lane, left) : 0);
      });
      if (lane == 0) {
        t.chunk = chunk;
        t.d = d;
        t.last = chunk == last;
        t.only_map = only_map;
        t.valid = min(total - base, int64_t{kRows});
        const bool plain = inside && !only_map && base + kRows <= total && left == 64;
        sh.tiles[s] = Tile{base * p.D + c0, d, plain ? 1 : 0};
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
      ++k;
    }
    // after a wait that ran out: no copy may be in flight when the CTA ends
    if (kFetch == kRowCopies) wait_copies();
    if (*static_cast<volatile int *>(&sh.broken))
      for (int i = max(k - kStages, 0); i < k; ++i)
        mbar_wait(smem_u32(&sh.full[i % kStages]), (i / kStages) & 1);
    return;
  }

  if (warp > kSlots) {
    // ---- chain ----
    for (int k = 0;; ++k) {
      const int s = k % kStages;
      const uint32_t parity = (k / kStages) & 1;
      if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.full[s]), parity, &sh.broken))) return;
      const Table<kRows> &tab = sh.tables[s];
      const int64_t chunk = tab.chunk;
      if (chunk < 0) return;
      const int64_t lane_ch = static_cast<int64_t>(tab.d) * 64 + 2 * lane, row_ch = static_cast<int64_t>(nt) * 64;
      const bool enters = !(tab.ends[1] >> 31) && !tab.last;  // the R behind the chunk matters
      const int64_t group = group_len == 1 ? chunk : chunk / kGroupLen;
      const int place = group_len == 1 ? 0 : kGroupLen - 1 - static_cast<int>(chunk % kGroupLen);
      const bool from_state = tab.ahead > place;  // the sequence goes on beyond the group
      const int before = from_state ? place : static_cast<int>(tab.ahead);
      const bool looks = enters && !tab.only_map, groups = group_len > 1;
      // the words that are looked at are those of chunks behind this one
      GDN_DCHECK(!looks || (before >= 0 && before < kGroupLen && (from_state || before >= 1) && chunk + before <= last &&
                            (!from_state || (group_len == 1 ? chunk + 1 : (chunk / kGroupLen + 1) * kGroupLen) <= last)));
      Words2 w[kGroupLen];
      auto src = [&](int j) {
        return j > 0 ? p.maps + (chunk + before - j + 1) * row_ch + lane_ch : states + (group + 1) * row_ch + lane_ch;
      };
      w[0] = looks && from_state ? try_words2(src(0)) : Words2{0, 0};
      if (groups) {
#pragma unroll
        for (int j = 1; j < kGroupLen; ++j) w[j] = looks && j <= before ? try_words2(src(j)) : Words2{0, 0};
      }
      uint64_t h = 0;
      if (!tab.only_map)
        h = load2_f32<kVec>(p.carries + chunk * groups128 * 128 + tab.d * 64, lane, 64);
      if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.mapped[s]), parity, &sh.broken) &&
                                       wait_phase(smem_u32(&sh.taken[s]), parity, &sh.broken)))
        return;
      float4 *own = &sh.own[0][lane];
      const float2 *rev = &sh.rev[0][lane];
      const uint32_t ends[2] = {tab.ends[0], tab.ends[1]}, starts[2] = {tab.starts[0], tab.starts[1]};
      const bool publishes = chunk > 0 && !tab.only_map && place == group_len - 1;
      uint64_t R = 0;
      auto down = [&](int i, uint64_t r) {  // R through slot i
        const float4 v = own[32 * i];
        const float2 q = rev[32 * i];
        const uint64_t Q = f2_pack(q.x, q.y);
        return mask_bits(ends, i * kTokW, kTokW) ? Q : f2_fma(f2_pack(v.x, v.y), r, Q);
      };
      if (looks) {
        if (groups) {
          await_words2<kGroupLen>(w, src, &sh.broken);
        } else if (from_state) {
          Words2 one[1] = {w[0]};
          await_words2<1>(one, src, &sh.broken);
          w[0] = one[0];
        }
        if (from_state) R = w[0].map().H;
        if (groups) {
#pragma unroll
          for (int j = 1; j < kGroupLen; ++j)
            if (j <= before) R = apply2(w[j].map(), R);
        }
      }
      uint64_t r[kSlots];
#pragma unroll
      for (int i = kSlots - 1; i >= 0; --i) {
        r[i] = R;
        R = down(i, R);
      }
      if (publishes) put_words2(states + group * row_ch + lane_ch, 0, R);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        const float4 v = own[32 * i];
        own[32 * i] = make_float4(f2_lo(h), f2_hi(h), f2_lo(r[i]), f2_hi(r[i]));
        const uint64_t y = f2_pack(v.z, v.w);
        h = mask_bits(starts, i * kTokW, kTokW) ? y : f2_fma(f2_pack(v.x, v.y), h, y);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.ready[s]));
    }
  }

  // ---- consumers ----
  const int row0 = warp * kTokW;
  // x, a, b and d_out of a row of a tile
  auto load = [&](int s, const Tile &tile, int i, uint64_t (&in)[3], uint64_t &o) {
    const int row = row0 + i;
    const unsigned char *stage = smem + s * S::kStage;
    const int64_t t = sh.tables[s].chunk * kRows + row, c0 = static_cast<int64_t>(tile.d) * 64;
    const unsigned char *src = stage + row * S::kPitch;
    if constexpr (kFetch == kRowCopies) src += row_offset<kElement>(p.d_out, p.do_stride, t, c0);
    o = fetch2<E, kVec>(src, lane).pair();
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      src = stage + S::kPlane + w * S::kInPlane + row * S::kInPitch;
      if constexpr (kFetch == kRowCopies) src += row_offset<kInElement>(input(w), input_stride(w), t, c0);
      if constexpr (kPacked) {
        const uint32_t q = kVec ? reinterpret_cast<const uint16_t *>(src)[lane]
                                : static_cast<uint32_t>(src[lane]) | static_cast<uint32_t>(src[lane + 32]) << 8;
        in[w] = dequantise2(q, sh.scales[s][w][row]);
      } else {
        in[w] = fetch2<E, kVec>(src, lane).pair();
      }
    }
  };
  auto initial = [&](const Table<kRows> &tab, int64_t c0, int i) {  // the state before a first token
    GDN_DCHECK(tab.start[row0 + i] >= 0 && tab.start[row0 + i] < p.s.N);
    return p.state != nullptr ? load2_f32<kVec>(p.state + tab.start[row0 + i] * p.D + c0, lane,
                                                static_cast<int>(min(p.D - c0, int64_t{64})))
                              : 0;
  };
  auto final = [&](const Table<kRows> &tab, int64_t c0, int i) {  // R behind a last token
    GDN_DCHECK(tab.end[row0 + i] >= 0 && tab.end[row0 + i] < p.s.N);
    return p.d_final != nullptr ? load2_f32<kVec>(p.d_final + tab.end[row0 + i] * p.D + c0, lane,
                                                  static_cast<int>(min(p.D - c0, int64_t{64})))
                                : 0;
  };
  int s = 0, turn = 0;
  uint32_t parity = 0;
  while (true) {
    if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.full[s]), parity, &sh.broken))) return;
    const Tile tile = sh.tiles[s];
    if (tile.d < 0) return;
    {
      // first pass
      const Table<kRows> &tab = sh.tables[s];
      const int64_t c0 = static_cast<int64_t>(tile.d) * 64;
      const Params2 par{load2_f32<kVec>(sh.params[s][0], lane, 64), load2_f32<kVec>(sh.params[s][1], lane, 64)};
      uint64_t P = f2_dup(1.f), y = 0, Q = 0, P_mid = 0, y_mid = 0;  // _mid: after half the slot
      auto row = [&](int i, bool edge, int valid, unsigned starts, unsigned ends, bool &ended) {
        uint64_t in[3], o;
        load(s, tile, i, in, o);
        const uint64_t w = f2_fma(in[1], f2_dup(kLog2e), par.dt), sp = softplus2(w, ex2_neg_abs(w));
        const uint64_t beta = sigmoid_pair(in[2]);
        sh.kept[warp][i][lane] = make_ulonglong2(sp, beta);
        uint64_t g = gate_of(par.c, sp), u = f2_mul(beta, in[0]);
        if (edge) {
          if (i >= valid) g = f2_dup(1.f), u = 0, o = 0;
          if ((starts >> i) & 1) y = initial(tab, c0, i);
        }
        P = f2_mul(P, g);
        y = f2_fma(g, y, u);
        if (!edge) {
          Q = f2_fma(P, o, Q);
        } else if (!ended) {
          if ((ends >> i) & 1) {
            o = f2_add(o, final(tab, c0, i));
            ended = true;
          }
          Q = f2_fma(P, o, Q);
        }
        if (i == kTokW / 2 - 1) P_mid = P, y_mid = y;
      };
      bool ended = false;
      if (tile.plain) {
#pragma unroll
        for (int i = 0; i < kTokW; ++i) row(i, false, kTokW, 0, 0, ended);
      } else {
        const int valid = static_cast<int>(max(int64_t{0}, min(int64_t{kTokW}, tab.valid - row0)));
        const unsigned starts = mask_bits(tab.starts, row0, kTokW), ends = mask_bits(tab.ends, row0, kTokW);
#pragma unroll 1
        for (int i = 0; i < kTokW; ++i) row(i, true, valid, starts, ends, ended);
      }
      sh.own[warp][lane] = make_float4(f2_lo(P), f2_hi(P), f2_lo(y), f2_hi(y));
      sh.rev[warp][lane] = make_float2(f2_lo(Q), f2_hi(Q));
      __syncwarp();
      const uint32_t mapped = smem_u32(&sh.mapped[s]);
      if (lane == 0) mbar_arrive(mapped);
      if (warp == turn) {
        const bool group_end = group_len == 1 || tab.chunk % kGroupLen == 0;
        if (tab.chunk > 0 && (!group_end || tab.only_map)) {
          if (!__all_sync(0xffffffffu, wait_phase(mapped, parity, &sh.broken))) return;
          auto map = [&](int i) {
            const float4 v = sh.own[i][lane];
            const float2 q = sh.rev[i][lane];
            return Map2{mask_bits(tab.ends, i * kTokW, kTokW) ? f2_dup(-1.f) : f2_pack(v.x, v.y), f2_pack(q.x, q.y)};
          };
          Map2 all = map(kSlots - 1);
#pragma unroll
          for (int i = kSlots - 2; i >= 0; --i) all = compose2(all, map(i));
          const int64_t at = c0 + 2 * lane;
          if (group_end)  // only_map: a sequence ends here, so the map is the R before it
            put_words2(states + (group_len == 1 ? tab.chunk : tab.chunk / kGroupLen) * nt * 64 + at, 0, all.H);
          else
            put_words2(p.maps + tab.chunk * nt * 64 + at, all.A, all.H);
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(smem_u32(&sh.taken[s]));
      }
      turn = turn + 1 == kSlots ? 0 : turn + 1;

      // second pass
      if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.ready[s]), parity, &sh.broken))) return;
      if (!tab.only_map) {
        const float4 in4 = sh.own[warp][lane];
        const uint64_t h_in = f2_pack(in4.x, in4.y);
        uint64_t R = f2_pack(in4.z, in4.w), sum_lg = 0, sum_da = 0;
        const int64_t at = tile.at + row0 * p.D;
        constexpr int kHalf = kTokW / 2;
        auto half = [&](int i0, bool edge, int valid, unsigned starts, unsigned ends, int left) {
          uint64_t g[kHalf], o[kHalf], beta[kHalf], xs[kHalf], ca[kHalf], cl[kHalf];
          uint64_t h = h_in;
          if (i0 > 0) {  // the state in the middle of the slot
            h = y_mid;
            if (!edge || !(starts & ((1u << kHalf) - 1u))) h = f2_fma(P_mid, h_in, h);
          }
#pragma unroll
          for (int j = 0; j < kHalf; ++j) {
            uint64_t in[3];
            load(s, tile, i0 + j, in, o[j]);
            if (edge && ((starts >> (i0 + j)) & 1)) h = initial(tab, c0, i0 + j);
            const ulonglong2 kept = sh.kept[warp][i0 + j][lane];
            const uint64_t sp = kept.x;
            beta[j] = kept.y;
            xs[j] = f2_mul(in[0], f2_fma(f2_mul(beta[j], f2_dup(-1.f)), beta[j], beta[j]));  // x beta (1 - beta)
            // sigmoid(z) = 2^(w - sp): z less softplus(z) is its logarithm (0 at
            // most; the difference of two infinities counts as that)
            const uint64_t w = f2_fma(in[1], f2_dup(kLog2e), par.dt), ls = f2_fma(sp, f2_dup(-1.f), w);
            const uint64_t sig = ex2_pair(f2_pack(fminf(f2_lo(ls), 0.f), fminf(f2_hi(ls), 0.f)));
            g[j] = gate_of(par.c, sp);
            const uint64_t gh = f2_mul(g[j], h), cgh = f2_mul(par.c, gh);  // -exp(A_log) g h_{t-1}
            h = f2_fma(g[j], h, f2_mul(beta[j], in[0]));
            ca[j] = f2_mul(cgh, sig);
            cl[j] = f2_mul(cgh, sp);
          }
#pragma unroll
          for (int j = kHalf - 1; j >= 0; --j) {
            const int i = i0 + j;
            if (edge) {
              if (i >= valid) continue;
              if ((ends >> i) & 1) R = final(tab, c0, i);
            }
            GDN_DCHECK(tab.chunk * kRows + row0 + i < total && (!edge || i < valid));
            const uint64_t dh = f2_add(o[j], R);
            R = f2_mul(g[j], dh);
            const uint64_t da = f2_mul(ca[j], dh);
            sum_da = f2_add(sum_da, da);
            sum_lg = f2_fma(cl[j], dh, sum_lg);  // dlg lg log2(e)
            store2<E, kVec>(static_cast<E *>(p.dx) + at + i * p.D, lane, left, f2_mul(beta[j], dh));
            store2<E, kVec>(static_cast<E *>(p.da) + at + i * p.D, lane, left, da);
            store2<E, kVec>(static_cast<E *>(p.db) + at + i * p.D, lane, left, f2_mul(xs[j], dh));
            if (edge && ((starts >> i) & 1) && p.d_state != nullptr)
              store2_f32<kVec>(p.d_state + tab.start[row0 + i] * p.D + c0, lane, left, R);
          }
        };
        if (tile.plain) {
          half(kHalf, false, kTokW, 0, 0, 64);
          half(0, false, kTokW, 0, 0, 64);
        } else {
          const int left = static_cast<int>(min(p.D - c0, int64_t{64}));
          const int valid = static_cast<int>(max(int64_t{0}, min(int64_t{kTokW}, tab.valid - row0)));
          const unsigned starts = mask_bits(tab.starts, row0, kTokW), ends = mask_bits(tab.ends, row0, kTokW);
#pragma unroll 1
          for (int i0 = kHalf; i0 >= 0; i0 -= kHalf) half(i0, true, valid, starts, ends, left);
        }
        constexpr float kLn2 = 0.6931471805599453f;
        __syncwarp();  // all lanes have read the warp's rows
        *reinterpret_cast<float4 *>(smem + s * S::kStage + warp * (S::kPlane / kSlots) + lane * 16) =
            make_float4(f2_lo(sum_lg) * kLn2, f2_hi(sum_lg) * kLn2, f2_lo(sum_da), f2_hi(sum_da));
        fence_async_smem();  // the next copy into this stage comes after
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.empty[s]));
    }
    if (++s == kStages) s = 0, parity ^= 1;
  }
}

// Sums the chunks' parts of the parameters' gradients [chunk][D up to 128s] in a
// fixed order: 32 threads of a channel take every 32nd chunk, then their sums
// are added.
__global__ void __launch_bounds__(1024)
recurrence_params_kernel(const float2 *partials, const Header *hdr, const Seqs s, int64_t D,
                         float *dA_log, float *ddt_bias) {
  __shared__ float2 part[32][33];
  if (hdr->bad) return;
  const int64_t total = s.total();
  const int64_t chunks = total > 0 ? (total - 1) / kRows + 1 : 0;
  const int64_t channel = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x, width = (D + 127) / 128 * 128;
  float2 v = make_float2(0.f, 0.f);
#pragma unroll 8
  for (int64_t c = threadIdx.y; c < chunks; c += 32) {
    const float2 q = partials[c * width + channel];
    v.x += q.x;
    v.y += q.y;
  }
  part[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0) {
    for (int i = 1; i < 32; ++i) v.x += part[i][threadIdx.x].x, v.y += part[i][threadIdx.x].y;
    if (channel < D) {
      dA_log[channel] = v.x;
      ddt_bias[channel] = v.y;
    }
  }
}

template <typename E, Fetch kFetch, bool kPacked>
cudaError_t launch_backward_t(Backward p, void *workspace, int sms, float *dA_log, float *ddt_bias,
                              cudaStream_t stream) {
  using S = BwdShape<E, kFetch, kPacked>;
  const int64_t nt = (p.D + 63) / 64, chunks = chunks_of(p.s.T);
  constexpr int smem = S::kStages * S::kStage + static_cast<int>(sizeof(BwdShared<S, kPacked>));
  static_assert(smem * S::kCtas <= 227 * 1024 - 1024 * (S::kCtas - 1), "CTAs of an SM share 228 KiB");
  if constexpr (kFetch == kTmaTile) {
    bool ok = make_row_map<E>(&p.to, p.d_out, p.D, p.s.T, p.do_stride, 64, kRows);
    if constexpr (kPacked) {
      const int64_t plane = p.s.T * p.D;
      ok = ok && make_row_map<uint8_t>(&p.tx, p.packed, p.D, p.s.T, p.D, 64, kRows) &&
           make_row_map<uint8_t>(&p.ta, p.packed + plane, p.D, p.s.T, p.D, 64, kRows) &&
           make_row_map<uint8_t>(&p.tb, p.packed + 2 * plane, p.D, p.s.T, p.D, 64, kRows);
    } else {
      ok = ok && make_row_map<E>(&p.tx, p.x, p.D, p.s.T, p.x_stride, 64, kRows) &&
           make_row_map<E>(&p.ta, p.a, p.D, p.s.T, p.a_stride, 64, kRows) &&
           make_row_map<E>(&p.tb, p.b, p.D, p.s.T, p.b_stride, 64, kRows);
    }
    if (!ok) return cudaErrorInvalidValue;
  }
  auto kernel = recurrence_backward_kernel<E, kFetch, kPacked>;
  static std::atomic<unsigned long long> allowed;
  if (cudaError_t e = allow_shared(kernel, smem, allowed)) return e;
  const Places w = places(workspace, p.s.T, p.D);
  p.hdr = static_cast<Header *>(workspace);
  p.maps = w.words;
  p.states = p.maps + chunks * nt * 64;
  p.dt = w.dt, p.c = w.c, p.first = w.first;
  const int64_t words = (chunks + (chunks + kGroupLen - 1) / kGroupLen) * nt * 64;
  const Prepared q{p.A_log,     p.dt_bias, w.dt,  w.c, p.D, w.first, chunks, kRows,
                   streams_for(nt, int64_t{sms} * S::kCtas), nt, int64_t{sms} * S::kCtas, true, nullptr, nullptr};
  if (cudaError_t e = launch_init(p.hdr, p.maps, words, p.s, q, stream)) return e;
  kernel<<<static_cast<unsigned>(min(chunks * nt, int64_t{sms} * S::kCtas)), S::kThreads, smem, stream>>>(p);
  if (cudaError_t e = cudaGetLastError()) return e;
  recurrence_params_kernel<<<static_cast<unsigned>(tiles_of(p.D) * 4), dim3(32, 32), 0, stream>>>(
      p.partials, p.hdr, p.s, p.D, dA_log, ddt_bias);
  return cudaGetLastError();
}

template <typename E>
cudaError_t launch_backward_e(const Backward &p, bool tma, void *workspace, int sms, float *dA_log, float *ddt_bias,
                              cudaStream_t stream) {
  if (p.packed != nullptr)
    return tma ? launch_backward_t<E, kTmaTile, true>(p, workspace, sms, dA_log, ddt_bias, stream)
               : launch_backward_t<E, kRowCopies, true>(p, workspace, sms, dA_log, ddt_bias, stream);
  return tma ? launch_backward_t<E, kTmaTile, false>(p, workspace, sms, dA_log, ddt_bias, stream)
             : launch_backward_t<E, kRowCopies, false>(p, workspace, sms, dA_log, ddt_bias, stream);
}

}  // namespace rec
}  // namespace gdn
