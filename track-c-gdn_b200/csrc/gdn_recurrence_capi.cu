// gdn_recurrence_capi.cu -- extern "C" entry points of the channelwise gated
// linear recurrence and the 8-bit checkpoints (declared in include/gdn_b200.h).
#include "../../include/gdn_b200.h"
#include "gdn_recurrence.cuh"

namespace {

using gdn::rec::chunks_of;
using gdn::rec::tiles_of;

constexpr int64_t kMaxTokens = int64_t{1} << 31;
constexpr int64_t kMaxSeqs = int64_t{1} << 24;

size_t type_size(int type) { return type == GDN_FP32 ? 4 : 2; }
bool known_type(int type) { return type == GDN_BF16 || type == GDN_FP16 || type == GDN_FP32; }

// Sizes that every recurrence call shares.
bool good_sizes(int type, int64_t T, int64_t N, int64_t D) {
  return known_type(type) && T >= 0 && T <= kMaxTokens && N >= 0 && N <= kMaxSeqs && D >= 1 &&
         D <= (int64_t{1} << 24) && chunks_of(T) <= INT32_MAX / tiles_of(D);
}

// Four-channel accesses need every row on a boundary of four elements.
bool vector_rows(const void *p, int type, int64_t stride) {
  return aligned(p, 4 * type_size(type)) && stride % 4 == 0;
}

bool bad_element_alignment(int type, std::initializer_list<const void *> ps) {
  for (const void *p : ps)
    if (p && !aligned(p, type_size(type))) return true;
  return false;
}

bool bad_f32_alignment(std::initializer_list<const void *> ps) {
  for (const void *p : ps)
    if (p && !aligned(p, 4)) return true;
  return false;
}

// Whether rows can be fetched by TMA: 16-byte rows and bases.
bool tma_rows(const void *p, int type, int64_t stride) {
  return aligned(p, 16) && stride * type_size(type) % 16 == 0 && stride > 0;
}

// Whether rows of D elements at p, `stride` elements apart, share memory with the
// dense [T, D] at q.
bool rows_overlap(const void *p, int64_t stride, const void *q, int type, int64_t T, int64_t D) {
  const size_t e = type_size(type);
  return p && q && T > 0 && overlap(p, ((T - 1) * stride + D) * e, q, static_cast<size_t>(T) * D * e);
}

// Memory that a call writes to or reads; nothing where the pointer is NULL.
struct Region {
  const void *p;
  size_t bytes;
};
bool meet(const Region &a, const Region &b) {
  return a.p && b.p && a.bytes && b.bytes && overlap(a.p, a.bytes, b.p, b.bytes);
}
// Whether an output shares memory with an input or with another output.
bool outputs_meet(std::initializer_list<Region> outs, std::initializer_list<Region> ins) {
  for (const Region *a = outs.begin(); a != outs.end(); ++a) {
    for (const Region &b : ins)
      if (meet(*a, b)) return true;
    for (const Region *b = outs.begin(); b != a; ++b)
      if (meet(*a, *b)) return true;
  }
  return false;
}

gdn::rec::Seqs sequences(const int64_t *cu, int64_t N, int64_t T, const int32_t *slots, int64_t pool) {
  return gdn::rec::Seqs{cu, N, T, N > 0 ? T / N : 0, slots, pool};
}

int run_forward(int type, const gdn::rec::Forward &p, void *workspace, int sms, cudaStream_t s) {
  const bool tma = p.s.T > 0 && p.s.T <= INT32_MAX && tma_rows(p.x, type, p.x_stride) &&
                   tma_rows(p.a, type, p.a_stride) && tma_rows(p.b, type, p.b_stride) && p.D % 4 == 0 &&
                   aligned(p.out, 8) && aligned(p.A_log, 8) && aligned(p.dt_bias, 8) && aligned(p.state, 8) &&
                   aligned(p.final, 8);
  const cudaError_t e = type == GDN_BF16   ? gdn::rec::launch_forward_e<__nv_bfloat16>(p, tma, workspace, sms, s)
                        : type == GDN_FP16 ? gdn::rec::launch_forward_e<__half>(p, tma, workspace, sms, s)
                                           : gdn::rec::launch_forward_e<float>(p, tma, workspace, sms, s);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // namespace

extern "C" {

size_t gdn_recurrence_workspace_bytes(int64_t total_tokens, int64_t channels) {
  if (!good_sizes(GDN_BF16, total_tokens, 1, channels)) return 0;
  return (gdn::rec::places(nullptr, total_tokens, channels).bytes + 1023) / 1024 * 1024;
}

size_t gdn_recurrence_carry_bytes(int64_t total_tokens, int64_t channels) {
  if (!good_sizes(GDN_BF16, total_tokens, 1, channels)) return 0;
  return gdn::rec::saved_bytes(total_tokens, channels);
}

size_t gdn_recurrence_packed_bytes(int64_t total_tokens, int64_t channels) {
  if (!good_sizes(GDN_BF16, total_tokens, 1, channels)) return 0;
  return 3 * static_cast<size_t>(total_tokens) * static_cast<size_t>(channels + tiles_of(channels));
}

size_t gdn_recurrence_backward_workspace_bytes(int64_t total_tokens, int64_t channels) {
  if (!good_sizes(GDN_BF16, total_tokens, 1, channels)) return 0;
  return gdn_recurrence_workspace_bytes(total_tokens, channels) +
         3 * gdn::rec::saved_bytes(total_tokens, channels);  // states, and two sums a channel
}

int gdn_recurrence_prefill(int type, const void *x, int64_t x_stride, const void *a, int64_t a_stride,
                           const void *b, int64_t b_stride, const float *A_log, const float *dt_bias,
                           const float *state, const int32_t *slots, int64_t pool_slots,
                           const int64_t *cu_seqlens, int64_t num_seqs, int64_t total_tokens,
                           int64_t channels, int zero_behind, void *out, float *final_state, float *carries,
                           void *packed, void *workspace, size_t workspace_bytes, void *stream) {
  if (!good_sizes(type, total_tokens, num_seqs, channels) || (slots && pool_slots < 1)) return GDN_ERR_BAD_SIZE;
  if (x_stride < 0 || a_stride < 0 || b_stride < 0) return GDN_ERR_BAD_SIZE;
  if (num_seqs == 0) return total_tokens == 0 ? GDN_OK : GDN_ERR_BAD_SIZE;
  if (!cu_seqlens && total_tokens % num_seqs != 0) return GDN_ERR_BAD_SIZE;
  if (!A_log || !dt_bias || !final_state || !workspace) return GDN_ERR_NULL_POINTER;
  if (slots && !state) return GDN_ERR_NULL_POINTER;
  if (total_tokens > 0 && (!x || !a || !b || !out)) return GDN_ERR_NULL_POINTER;
  if (bad_element_alignment(type, {x, a, b, out}) ||
      bad_f32_alignment({A_log, dt_bias, state, final_state, slots}) ||
      (cu_seqlens && !aligned(cu_seqlens, 8)) || (carries && !aligned(carries, 16)) ||
      (packed && !aligned(packed, 16)))
    return GDN_ERR_MISALIGNED;
  if (!aligned(workspace, 1024) || workspace_bytes < gdn_recurrence_workspace_bytes(total_tokens, channels))
    return GDN_ERR_WORKSPACE;
  const size_t states = static_cast<size_t>(slots ? pool_slots : num_seqs) * channels * 4;
  if (state && state != final_state && overlap(state, states, final_state, states)) return GDN_ERR_ALIASING;
  // rows are read again after others have been written (chunks cut by streams)
  if (rows_overlap(x, x_stride, out, type, total_tokens, channels) ||
      rows_overlap(a, a_stride, out, type, total_tokens, channels) ||
      rows_overlap(b, b_stride, out, type, total_tokens, channels))
    return GDN_ERR_ALIASING;
  const size_t outs = static_cast<size_t>(total_tokens) * channels * type_size(type);
  if (outputs_meet({{out, outs},
                    {final_state, states},
                    {carries, gdn_recurrence_carry_bytes(total_tokens, channels)},
                    {packed, gdn_recurrence_packed_bytes(total_tokens, channels)},
                    {workspace, gdn_recurrence_workspace_bytes(total_tokens, channels)}},
                   {}) ||
      (state != final_state && meet({state, states}, {out, outs})))
    return GDN_ERR_ALIASING;
  int sms = 0;
  if (int st = check_device(&sms)) return st;
  gdn::rec::Forward p{};
  p.x = x, p.a = a, p.b = b;
  p.x_stride = x_stride, p.a_stride = a_stride, p.b_stride = b_stride;
  p.A_log = A_log, p.dt_bias = dt_bias, p.state = state;
  p.s = sequences(cu_seqlens, num_seqs, total_tokens, slots, pool_slots);
  p.D = channels, p.zero_behind = zero_behind && cu_seqlens && total_tokens > 0;
  p.out = out, p.final = final_state, p.carries = carries, p.packed = static_cast<uint8_t *>(packed);
  return run_forward(type, p, workspace, sms, static_cast<cudaStream_t>(stream));
}

int gdn_recurrence_backward(int type, const void *x, int64_t x_stride, const void *a, int64_t a_stride,
                            const void *b, int64_t b_stride, const void *packed, const float *A_log,
                            const float *dt_bias, const float *state, const int64_t *cu_seqlens,
                            int64_t num_seqs, int64_t total_tokens, int64_t channels, int zero_behind,
                            const void *d_out, int64_t d_out_stride, const float *d_final_state,
                            const float *carries, void *dx, void *da, void *db, float *dA_log, float *ddt_bias, float *d_state,
                            void *workspace, size_t workspace_bytes, void *stream) {
  if (!good_sizes(type, total_tokens, num_seqs, channels)) return GDN_ERR_BAD_SIZE;
  if (x_stride < 0 || a_stride < 0 || b_stride < 0 || d_out_stride < 0) return GDN_ERR_BAD_SIZE;
  if (num_seqs == 0 && total_tokens != 0) return GDN_ERR_BAD_SIZE;
  if (!cu_seqlens && num_seqs > 0 && total_tokens % num_seqs != 0) return GDN_ERR_BAD_SIZE;
  if (!A_log || !dt_bias || !dA_log || !ddt_bias || !workspace) return GDN_ERR_NULL_POINTER;
  if (total_tokens > 0 && (!d_out || !dx || !da || !db)) return GDN_ERR_NULL_POINTER;
  // the inputs, or their 8-bit form with the states that the forward saved
  if (total_tokens > 0 && (packed ? !carries : !x || !a || !b)) return GDN_ERR_NULL_POINTER;
  if (bad_element_alignment(type, {x, a, b, d_out, dx, da, db}) ||
      bad_f32_alignment({A_log, dt_bias, state, d_final_state, dA_log, ddt_bias, d_state}) ||
      (cu_seqlens && !aligned(cu_seqlens, 8)) || (carries && !aligned(carries, 16)) ||
      (packed && !aligned(packed, 16)))
    return GDN_ERR_MISALIGNED;
  if (!aligned(workspace, 1024) ||
      workspace_bytes < gdn_recurrence_backward_workspace_bytes(total_tokens, channels))
    return GDN_ERR_WORKSPACE;
  const size_t states = static_cast<size_t>(num_seqs) * channels * 4;
  if (d_state && ((state && overlap(state, states, d_state, states)) ||
                  (d_final_state && overlap(d_final_state, states, d_state, states))))
    return GDN_ERR_ALIASING;
  for (void *g : {dx, da, db}) {
    if (rows_overlap(d_out, d_out_stride, g, type, total_tokens, channels)) return GDN_ERR_ALIASING;
    if (!packed && (rows_overlap(x, x_stride, g, type, total_tokens, channels) ||
                    rows_overlap(a, a_stride, g, type, total_tokens, channels) ||
                    rows_overlap(b, b_stride, g, type, total_tokens, channels)))
      return GDN_ERR_ALIASING;
  }
  const size_t rows = static_cast<size_t>(total_tokens) * channels * type_size(type);
  if (outputs_meet({{dx, rows},
                    {da, rows},
                    {db, rows},
                    {d_state, states},
                    {workspace, gdn_recurrence_backward_workspace_bytes(total_tokens, channels)}},
                   {{state, states},
                    {d_final_state, states},
                    {carries, gdn_recurrence_carry_bytes(total_tokens, channels)},
                    {packed, gdn_recurrence_packed_bytes(total_tokens, channels)}}))
    return GDN_ERR_ALIASING;
  int sms = 0;
  if (int st = check_device(&sms)) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const gdn::rec::Seqs seqs = sequences(cu_seqlens, num_seqs, total_tokens, nullptr, 0);
  if (num_seqs == 0) {
    const cudaError_t e0 = cudaMemsetAsync(dA_log, 0, channels * 4, s);
    const cudaError_t e1 = cudaMemsetAsync(ddt_bias, 0, channels * 4, s);
    return e0 == cudaSuccess && e1 == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
  }
  const bool tma =
      total_tokens > 0 && total_tokens <= INT32_MAX && channels % 4 == 0 &&
      (packed ? channels % 16 == 0
              : tma_rows(x, type, x_stride) && tma_rows(a, type, a_stride) && tma_rows(b, type, b_stride)) &&
      tma_rows(d_out, type, d_out_stride) && aligned(dx, 8) && aligned(da, 8) && aligned(db, 8) &&
      aligned(A_log, 8) && aligned(dt_bias, 8) && aligned(state, 8) && aligned(d_final_state, 8) &&
      aligned(d_state, 8);
  char *extra = static_cast<char *>(workspace) + gdn_recurrence_workspace_bytes(total_tokens, channels);
  float *saved = reinterpret_cast<float *>(extra);
  if (!carries) {
    // the states that enter the chunks, by the forward without its outputs
    gdn::rec::Forward f{};
    f.x = x, f.a = a, f.b = b;
    f.x_stride = x_stride, f.a_stride = a_stride, f.b_stride = b_stride;
    f.A_log = A_log, f.dt_bias = dt_bias, f.state = state, f.s = seqs, f.D = channels, f.carries = saved;
    if (int st = run_forward(type, f, workspace, sms, s)) return st;
  }
  gdn::rec::Backward p{};
  p.x = x, p.a = a, p.b = b, p.d_out = d_out;
  p.x_stride = x_stride, p.a_stride = a_stride, p.b_stride = b_stride, p.do_stride = d_out_stride;
  p.packed = static_cast<const uint8_t *>(packed);
  p.A_log = A_log, p.dt_bias = dt_bias, p.state = state, p.d_final = d_final_state;
  p.carries = carries ? carries : saved;
  p.s = seqs, p.D = channels, p.zero_behind = zero_behind && cu_seqlens && total_tokens > 0;
  p.dx = dx, p.da = da, p.db = db, p.d_state = d_state;
  p.partials = reinterpret_cast<float2 *>(extra + gdn::rec::saved_bytes(total_tokens, channels));
  const cudaError_t e =
      type == GDN_BF16   ? gdn::rec::launch_backward_e<__nv_bfloat16>(p, tma, workspace, sms, dA_log, ddt_bias, s)
      : type == GDN_FP16 ? gdn::rec::launch_backward_e<__half>(p, tma, workspace, sms, dA_log, ddt_bias, s)
                         : gdn::rec::launch_backward_e<float>(p, tma, workspace, sms, dA_log, ddt_bias, s);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

int gdn_recurrence_decode(int type, const void *x, int64_t x_stride, const void *a, int64_t a_stride,
                          const void *b, int64_t b_stride, const float *A_log, const float *dt_bias,
                          const float *state, const int32_t *slots, int64_t pool_slots, int64_t batch,
                          int64_t num_tokens, int64_t channels, void *out, float *new_state,
                          float *intermediate_states, void *stream) {
  if (!known_type(type) || batch < 0 || batch > kMaxSeqs || num_tokens < 1 ||
      num_tokens > GDN_DECODE_MTP_MAX_TOKENS || channels < 1 || channels > (int64_t{1} << 24) ||
      batch * tiles_of(channels) > INT32_MAX || (slots && pool_slots < 1) || x_stride < 0 || a_stride < 0 ||
      b_stride < 0)
    return GDN_ERR_BAD_SIZE;
  if (batch == 0) return GDN_OK;
  if (!x || !a || !b || !A_log || !dt_bias || !out || !new_state || (slots && !state))
    return GDN_ERR_NULL_POINTER;
  if (bad_element_alignment(type, {x, a, b, out}) ||
      bad_f32_alignment({A_log, dt_bias, state, new_state, intermediate_states, slots}))
    return GDN_ERR_MISALIGNED;
  const size_t states = static_cast<size_t>(slots ? pool_slots : batch) * channels * 4;
  const int64_t rows = batch * num_tokens;
  const size_t inter = static_cast<size_t>(rows) * channels * 4, outs = static_cast<size_t>(rows) * channels * type_size(type);
  if ((state && state != new_state && overlap(state, states, new_state, states)) ||
      (intermediate_states && ((state && overlap(state, states, intermediate_states, inter)) ||
                               overlap(new_state, states, intermediate_states, inter))))
    return GDN_ERR_ALIASING;
  if (overlap(out, outs, new_state, states) || (state && overlap(out, outs, state, states)) ||
      (intermediate_states && overlap(out, outs, intermediate_states, inter)))
    return GDN_ERR_ALIASING;
  // `out` in the very place of an input: a lane reads what it then writes
  const void *const inputs[3] = {x, a, b};
  const int64_t strides[3] = {x_stride, a_stride, b_stride};
  for (int i = 0; i < 3; ++i) {
    const size_t bytes = static_cast<size_t>((rows - 1) * strides[i] + channels) * type_size(type);
    const bool same = out == inputs[i] && (strides[i] == channels || rows == 1);
    if ((!same && overlap(inputs[i], bytes, out, outs)) || overlap(inputs[i], bytes, new_state, states) ||
        (intermediate_states && overlap(inputs[i], bytes, intermediate_states, inter)))
      return GDN_ERR_ALIASING;
  }
  if (int st = check_device(nullptr)) return st;
  gdn::rec::Decode p{x, a, b, x_stride, a_stride, b_stride, A_log, dt_bias, state, slots, pool_slots, batch,
                     channels, static_cast<int>(num_tokens), out, new_state, intermediate_states};
  const bool vec = channels % 4 == 0 && vector_rows(x, type, x_stride) && vector_rows(a, type, a_stride) &&
                   vector_rows(b, type, b_stride) && vector_rows(out, type, channels) && aligned(A_log, 16) &&
                   aligned(dt_bias, 16) && (!state || aligned(state, 16)) && aligned(new_state, 16) &&
                   (!intermediate_states || aligned(intermediate_states, 16));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = type == GDN_BF16   ? gdn::rec::launch_decode_e<__nv_bfloat16>(p, vec, s)
                        : type == GDN_FP16 ? gdn::rec::launch_decode_e<__half>(p, vec, s)
                                           : gdn::rec::launch_decode_e<float>(p, vec, s);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // extern "C"

namespace {

int checkpoint_call(int type, const gdn_checkpoint_tensor *tensors, int count, bool unpack, void *stream) {
  if (!known_type(type) || count < 0 || count > GDN_CHECKPOINT_MAX_TENSORS) return GDN_ERR_BAD_SIZE;
  if (count > 0 && !tensors) return GDN_ERR_NULL_POINTER;
  using gdn::rec::kGroupValues;
  gdn::rec::Pack p{};
  bool vec = true;
  int64_t warps = 0;
  for (int i = 0; i < count; ++i) {
    const gdn_checkpoint_tensor &t = tensors[i];
    if (t.rows < 0 || t.cols < 0 || t.inner < 1 || t.rows > INT32_MAX || t.inner > INT32_MAX || t.cols > INT32_MAX)
      return GDN_ERR_BAD_SIZE;
    if (t.rows == 0 || t.cols == 0) continue;
    if (!t.data || !t.values || !t.scales) return GDN_ERR_NULL_POINTER;
    if (!aligned(t.data, type_size(type))) return GDN_ERR_MISALIGNED;
    const int64_t groups = (t.cols + kGroupValues - 1) / kGroupValues, items = t.rows * groups;
    if (items > INT32_MAX) return GDN_ERR_BAD_SIZE;
    gdn::rec::PackTensor &k = p.t[p.count++];
    k.data = t.data;
    k.values = static_cast<uint8_t *>(t.values), k.scales = static_cast<uint8_t *>(t.scales);
    k.inner = static_cast<uint32_t>(t.inner), k.outer_stride = t.outer_stride, k.inner_stride = t.inner_stride;
    k.cols = t.cols, k.groups = static_cast<uint32_t>(groups), k.items = static_cast<uint32_t>(items);
    k.first = static_cast<uint32_t>(warps);
    warps += (items + gdn::rec::kItems - 1) / gdn::rec::kItems;
    const bool dense = unpack || t.rows == 1 ||
                       ((t.inner == 1 || t.inner_stride == t.cols) && t.outer_stride == t.inner * t.cols);
    k.flat = t.cols % kGroupValues == 0 && dense && (!unpack || (aligned(t.data, 16) && aligned(t.values, 8)));
    vec = vec && t.cols % 4 == 0 && aligned(t.data, 4 * type_size(type)) && aligned(t.values, 4) &&
          (unpack || (t.outer_stride % 4 == 0 && t.inner_stride % 4 == 0));
  }
  if (warps == 0) return GDN_OK;
  if (warps > INT32_MAX) return GDN_ERR_BAD_SIZE;
  if (int st = check_device(nullptr)) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t w = static_cast<uint32_t>(warps);
  const cudaError_t e = type == GDN_BF16   ? gdn::rec::launch_checkpoint_e<__nv_bfloat16>(p, w, vec, unpack, s)
                        : type == GDN_FP16 ? gdn::rec::launch_checkpoint_e<__half>(p, w, vec, unpack, s)
                                           : gdn::rec::launch_checkpoint_e<float>(p, w, vec, unpack, s);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int gdn_checkpoint_pack(int type, const gdn_checkpoint_tensor *tensors, int count, void *stream) {
  return checkpoint_call(type, tensors, count, false, stream);
}

int gdn_checkpoint_unpack(int type, const gdn_checkpoint_tensor *tensors, int count, void *stream) {
  return checkpoint_call(type, tensors, count, true, stream);
}

}  // extern "C"
