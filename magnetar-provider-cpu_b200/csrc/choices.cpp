// C ABI of the operators whose rows choose what they meet: adapters, packed
// experts and sampled tokens (argument checks; the kernels are in adapters.cu,
// experts.cu and sample.cu).
#include <cuda_runtime.h>

#include "../../include/magnetar_b200.h"
#include "api_internal.h"
#include "kernels.h"

namespace mgb {
namespace {

bool aligned(const void *p, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Element counts stay far inside 64 bits: no single extent, product of two
// extents or buffer passes 2^48 values.
constexpr uint64_t MAX_VALUES = 1ull << 48;
bool too_large(uint64_t a, uint64_t b, uint64_t c = 1) {
  if (a == 0 || b == 0 || c == 0) return false;
  if (a > MAX_VALUES || b > MAX_VALUES / a) return true;
  return c > MAX_VALUES / (a * b);
}

mgb_status check_workspace(const void *workspace, uint64_t have, uint64_t need) {
  if (!need) return MGB_OK;
  if (have < need || !workspace)
    return fail(MGB_INVALID_ARGUMENT, "workspace has %llu bytes, the call needs %llu",
                (unsigned long long)(workspace ? have : 0), (unsigned long long)need);
  if (!aligned(workspace, 16)) return fail(MGB_INVALID_ARGUMENT, "workspace is not 16-byte aligned");
  return MGB_OK;
}

// Whether two buffers of f32 values share any of them.
bool overlap(const float *a, uint64_t a_len, const float *b, uint64_t b_len) {
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  return a0 < b0 + b_len * 4 && b0 < a0 + a_len * 4;
}

uint64_t element_bytes(int32_t dtype) { return dtype == MGB_DTYPE_F32 ? 4 : 2; }

// The descriptor alone and m (the size queries and the calls).
mgb_status check_adapters(const mgb_adapters *ad, uint64_t m) {
  if (!ad) return fail(MGB_INVALID_ARGUMENT, "null adapter descriptor");
  if (ad->dtype != MGB_DTYPE_F32 && ad->dtype != MGB_DTYPE_F16 && ad->dtype != MGB_DTYPE_BF16)
    return fail(MGB_DTYPE_UNSUPPORTED, "adapters of dtype %d are not supported", ad->dtype);
  if (!ad->count || !ad->rank || !ad->k || !ad->n)
    return fail(MGB_INVALID_ARGUMENT, "adapters need count, rank, k and n of at least 1");
  if (ad->rank > MGB_MAX_ADAPTER_RANK)
    return fail(MGB_INVALID_ARGUMENT, "adapter rank %llu is above %d", (unsigned long long)ad->rank,
                MGB_MAX_ADAPTER_RANK);
  // ids are f32: whole numbers up to 2^24 are exact
  if (ad->count > (1u << 24) || m > (1u << 24) || ad->k > (1u << 30) || ad->n > (1u << 30) ||
      too_large(ad->count, ad->rank, ad->k) || too_large(ad->count, ad->rank, ad->n) ||
      too_large(m, ad->k) || too_large(m, ad->n))
    return fail(MGB_INVALID_ARGUMENT, "adapter sizes are too large");
  return MGB_OK;
}

mgb_status check_adapters_call(const mgb_adapters *ad, const float *ids, const float *x, uint64_t m,
                               const float *base, const float *y, const uint32_t *bad) {
  mgb_status s = check_adapters(ad, m);
  if (s != MGB_OK || !m) return s;
  if (!ad->a || !ad->b || !ids || !x || !y) return fail(MGB_INVALID_ARGUMENT, "null device pointer");
  const uint64_t e = element_bytes(ad->dtype);
  if (!aligned(ad->a, e) || !aligned(ad->b, e) || !aligned(ad->scales, 4) || !aligned(ids, 4) ||
      !aligned(x, 4) || !aligned(base, 4) || !aligned(y, 4) || !aligned(bad, 4))
    return fail(MGB_INVALID_ARGUMENT, "a device pointer is not aligned to its element size");
  return MGB_OK;
}

mgb_status check_experts(const mgb_experts *ex, uint64_t m, uint64_t top_k) {
  if (!ex) return fail(MGB_INVALID_ARGUMENT, "null expert descriptor");
  for (int32_t f : {ex->gate_up_format, ex->down_format})
    if (!format_supported(f))
      return fail(MGB_UNSUPPORTED, "packed format %d is not executed by this Provider", f);
  if (!ex->experts || ex->experts > MGB_MOE_MAX_EXPERTS)
    return fail(MGB_INVALID_ARGUMENT, "%llu experts, expected 1 to %d",
                (unsigned long long)ex->experts, MGB_MOE_MAX_EXPERTS);
  if (ex->hidden > MGB_MOE_MAX_WIDTH || ex->ffn > MGB_MOE_MAX_WIDTH || too_large(ex->experts, ex->hidden, ex->ffn))
    return fail(MGB_INVALID_ARGUMENT, "expert sizes are too large");
  mgb_status s = check_packed_shape(ex->gate_up_format, ex->experts * ex->ffn, ex->hidden);
  if (s == MGB_OK) s = check_packed_shape(ex->down_format, ex->experts * ex->hidden, ex->ffn);
  if (s != MGB_OK) return s;
  if (m > MGB_MOE_MAX_TOKENS)
    return fail(MGB_INVALID_ARGUMENT, "%llu tokens, at most %d are taken in one call",
                (unsigned long long)m, MGB_MOE_MAX_TOKENS);
  if (!top_k || top_k > MGB_MOE_MAX_TOP_K)
    return fail(MGB_INVALID_ARGUMENT, "top_k %llu, expected 1 to %d", (unsigned long long)top_k,
                MGB_MOE_MAX_TOP_K);
  // Stages of 128 rows by at least 128 columns are counted in 32 bits.  Gate and up have
  // two of them a block, but a pass of its own for more than half of the slots needs that
  // many experts: above 2^30 blocks of 2^14 weights, more than a GPU holds.
  const uint64_t blocks = (ex->hidden / 128 + 1) * (ex->ffn / 128 + 1);
  if (m * top_k * blocks >= (1ull << 31))
    return fail(MGB_INVALID_ARGUMENT, "expert sizes are too large for %llu tokens",
                (unsigned long long)m);
  return MGB_OK;
}

mgb_status check_experts_call(const mgb_experts *ex, const float *x, uint64_t m, const float *ids,
                              const float *weights, uint64_t top_k, const float *addend,
                              const float *y, const uint32_t *bad) {
  mgb_status s = check_experts(ex, m, top_k);
  if (s != MGB_OK || !m) return s;
  if (!ex->gate || !ex->up || !ex->down || !x || !ids || !weights || !y)
    return fail(MGB_INVALID_ARGUMENT, "null device pointer");
  if (!aligned(ex->gate, 16) || !aligned(ex->up, 16) || !aligned(ex->down, 16))
    return fail(MGB_INVALID_ARGUMENT, "packed expert pointers must be 16-byte aligned");
  if (!aligned(x, 16)) return fail(MGB_INVALID_ARGUMENT, "activation pointer is not 16-byte aligned");
  if (!aligned(ids, 4) || !aligned(weights, 4) || !aligned(addend, 4) || !aligned(y, 4) ||
      !aligned(bad, 4))
    return fail(MGB_INVALID_ARGUMENT, "a device pointer is not aligned to its element size");
  return MGB_OK;
}

mgb_status check_route(const float *router, uint64_t experts, uint64_t hidden, const float *x,
                       uint64_t m, uint64_t top_k) {
  if (!experts || experts > MGB_MOE_MAX_EXPERTS)
    return fail(MGB_INVALID_ARGUMENT, "%llu experts, expected 1 to %d", (unsigned long long)experts,
                MGB_MOE_MAX_EXPERTS);
  if (!hidden || hidden > MGB_MOE_MAX_WIDTH) return fail(MGB_INVALID_ARGUMENT, "hidden %llu is out of range", (unsigned long long)hidden);
  if (m > MGB_MOE_MAX_TOKENS)
    return fail(MGB_INVALID_ARGUMENT, "%llu tokens, at most %d are taken in one call",
                (unsigned long long)m, MGB_MOE_MAX_TOKENS);
  if (!top_k || top_k > MGB_MOE_MAX_TOP_K || top_k > experts)
    return fail(MGB_INVALID_ARGUMENT, "top_k %llu, expected 1 to %llu", (unsigned long long)top_k,
                (unsigned long long)(experts < MGB_MOE_MAX_TOP_K ? experts : MGB_MOE_MAX_TOP_K));
  if (m && (!router || !x)) return fail(MGB_INVALID_ARGUMENT, "null device pointer");
  if (!aligned(router, 4) || !aligned(x, 4))
    return fail(MGB_INVALID_ARGUMENT, "a device pointer is not aligned to its element size");
  return MGB_OK;
}

// The device error word of the current device (bounded waits that give up).
int *error_word() {
  int dev = 0;
  cudaGetDevice(&dev);
  return device_error_flag(dev);
}

uint64_t round16(uint64_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace
}  // namespace mgb

using namespace mgb;

extern "C" {

uint64_t mgb_adapters_workspace_bytes(const mgb_adapters *adapters, uint64_t m) {
  return check_adapters(adapters, m) == MGB_OK ? adapters_scratch_bytes(*adapters, m) : 0;
}

mgb_status mgb_adapters_add(const mgb_adapters *adapters, const float *ids, const float *x,
                            uint64_t m, const float *base, float *y, uint32_t *bad,
                            void *workspace, uint64_t workspace_bytes, void *stream) {
  mgb_status s = check_adapters_call(adapters, ids, x, m, base, y, bad);
  if (s == MGB_OK) s = check_workspace(workspace, workspace_bytes, adapters_scratch_bytes(*adapters, m));
  if (s != MGB_OK) return s;
  // (other rows' x and base are still read while a row's y is written)
  const uint64_t n = adapters->n;
  if (overlap(x, m * adapters->k, y, m * n) || (base && base != y && overlap(base, m * n, y, m * n)))
    return fail(MGB_INVALID_ARGUMENT, "y overlaps x, or base without being it");
  cudaError_t e = launch_adapters(*adapters, ids, x, m, base, y, bad, workspace,
                                  static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MGB_OK : cuda_fail(e, "adapter launch");
}

uint64_t mgb_qmatmul_adapters_workspace_bytes(int32_t format, uint64_t m, uint64_t n, uint64_t k,
                                              const mgb_adapters *adapters) {
  if (check_adapters(adapters, m) != MGB_OK) return 0;
  const uint64_t a = adapters_scratch_bytes(*adapters, m), q = qmatmul_scratch_bytes(format, m, n, k);
  return a > q ? a : q;
}

mgb_status mgb_qmatmul_adapters(int32_t format, const void *w, uint64_t n, uint64_t k,
                                const float *x, uint64_t m, float *y, const float *addend,
                                uint64_t addend_len, const mgb_adapters *adapters,
                                const float *ids, uint32_t *bad, void *workspace,
                                uint64_t workspace_bytes, void *stream) {
  mgb_status s = check_adapters_call(adapters, ids, x, m, y, y, bad);
  if (s != MGB_OK) return s;
  if (adapters->k != k || adapters->n != n)
    return fail(MGB_INVALID_ARGUMENT,
                "adapters of %llu inputs and %llu outputs beside a projection of %llu and %llu",
                (unsigned long long)adapters->k, (unsigned long long)adapters->n,
                (unsigned long long)k, (unsigned long long)n);
  s = check_workspace(workspace, workspace_bytes, adapters_scratch_bytes(*adapters, m));
  if (s == MGB_OK)
    s = mgb_qmatmul(format, w, n, k, x, m, y, addend, addend_len, workspace, workspace_bytes, stream);
  if (s != MGB_OK) return s;
  cudaError_t e = launch_adapters(*adapters, ids, x, m, y, y, bad, workspace,
                                  static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MGB_OK : cuda_fail(e, "adapter launch");
}

// (routing and sampling need no scratch)
uint64_t mgb_moe_route_workspace_bytes(uint64_t, uint64_t, uint64_t) { return 0; }

// The experts' scratch, then room for mgb_moe_layer's ids and weights.
uint64_t mgb_moe_workspace_bytes(const mgb_experts *experts, uint64_t m, uint64_t top_k) {
  if (check_experts(experts, m, top_k) != MGB_OK) return 0;
  return round16(moe_experts_scratch_bytes(*experts, m, top_k)) + 2 * round16(m * top_k * 4);
}

mgb_status mgb_moe_route(const float *router, uint64_t experts, uint64_t hidden, const float *x,
                         uint64_t m, uint64_t top_k, int32_t normalize, float scale, float *ids,
                         float *weights, void *, uint64_t, void *stream) {
  mgb_status s = check_route(router, experts, hidden, x, m, top_k);
  if (s == MGB_OK && m && (!ids || !weights)) s = fail(MGB_INVALID_ARGUMENT, "null device pointer");
  if (s == MGB_OK && (!aligned(ids, 4) || !aligned(weights, 4)))
    s = fail(MGB_INVALID_ARGUMENT, "a device pointer is not aligned to its element size");
  if (s != MGB_OK) return s;
  cudaError_t e = launch_moe_route(router, experts, hidden, x, m, top_k, normalize != 0, scale, ids,
                                   weights, nullptr, nullptr, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MGB_OK : cuda_fail(e, "routing launch");
}

mgb_status mgb_moe_experts(const mgb_experts *experts, const float *x, uint64_t m,
                           const float *ids, const float *weights, uint64_t top_k,
                           const float *addend, float *y, uint32_t *bad, void *workspace,
                           uint64_t workspace_bytes, void *stream) {
  mgb_status s = check_experts_call(experts, x, m, ids, weights, top_k, addend, y, bad);
  if (s == MGB_OK)
    s = check_workspace(workspace, workspace_bytes, moe_experts_scratch_bytes(*experts, m, top_k));
  if (s != MGB_OK) return s;
  cudaError_t e = launch_moe_experts(*experts, x, m, ids, weights, top_k, addend, y, bad, workspace,
                                     false, error_word(), static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MGB_OK : cuda_fail(e, "expert launch");
}

mgb_status mgb_moe_layer(const mgb_experts *experts, const float *router, const float *x,
                         uint64_t m, uint64_t top_k, int32_t normalize, float scale,
                         const float *addend, float *y, float *ids, float *weights,
                         void *workspace, uint64_t workspace_bytes, void *stream) {
  mgb_status s = check_experts(experts, m, top_k);
  if (s == MGB_OK) s = check_route(router, experts->experts, experts->hidden, x, m, top_k);
  if (s == MGB_OK)
    s = check_workspace(workspace, workspace_bytes, mgb_moe_workspace_bytes(experts, m, top_k));
  if (s != MGB_OK) return s;
  uint8_t *own = static_cast<uint8_t *>(workspace) +
                 round16(moe_experts_scratch_bytes(*experts, m, top_k));
  if (!ids) ids = reinterpret_cast<float *>(own);
  if (!weights) weights = reinterpret_cast<float *>(own + round16(m * top_k * 4));
  s = check_experts_call(experts, x, m, ids, weights, top_k, addend, y, nullptr);
  if (s != MGB_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_moe_route(router, experts->experts, experts->hidden, x, m, top_k,
                                   normalize != 0, scale, ids, weights, experts, workspace, st);
  if (e != cudaSuccess) return cuda_fail(e, "routing launch");
  e = launch_moe_experts(*experts, x, m, ids, weights, top_k, addend, y, nullptr, workspace, true,
                         error_word(), st);
  return e == cudaSuccess ? MGB_OK : cuda_fail(e, "expert launch");
}

uint64_t mgb_sample_workspace_bytes(uint64_t, uint64_t) { return 0; }

mgb_status mgb_sample(const float *logits, uint64_t rows, uint64_t vocab, uint64_t ld,
                      const float *temperature, const float *top_k, const float *top_p,
                      const float *min_p, const float *uniform, float *ids, float *logprob,
                      uint32_t *kept, void *, uint64_t, void *stream) {
  if (!vocab || vocab > MGB_SAMPLE_MAX_VOCAB)
    return fail(MGB_INVALID_ARGUMENT, "vocabulary of %llu tokens, expected 1 to %u",
                (unsigned long long)vocab, MGB_SAMPLE_MAX_VOCAB);
  if (ld < vocab)
    return fail(MGB_INVALID_ARGUMENT, "row stride %llu is below the vocabulary size %llu",
                (unsigned long long)ld, (unsigned long long)vocab);
  if (rows > (1ull << 31) || too_large(rows, ld)) return fail(MGB_INVALID_ARGUMENT, "too many rows");
  if (rows && !logits) return fail(MGB_INVALID_ARGUMENT, "null device pointer");
  for (const void *p : {(const void *)logits, (const void *)temperature, (const void *)top_k,
                        (const void *)top_p, (const void *)min_p, (const void *)uniform,
                        (const void *)ids, (const void *)logprob, (const void *)kept})
    if (!aligned(p, 4))
      return fail(MGB_INVALID_ARGUMENT, "a device pointer is not aligned to its element size");
  if (!rows) return MGB_OK;
  const SampleArgs a{logits, rows,  vocab,   ld,  temperature, top_k,
                     top_p,  min_p, uniform, ids, logprob,     kept};
  cudaError_t e = launch_sample(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MGB_OK : cuda_fail(e, "sampling launch");
}

}  // extern "C"
