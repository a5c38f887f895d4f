// Attention of a chunk of new tokens over the paged K/V pool, bf16 or e4m3 (sm_100a).
// Semantics: include/mac_b200_chunk.h.
#include <cuda_bf16.h>

#include <cmath>

#include "mac_b200_common.h"
#include "mac_b200_kv8.cuh"

#include "../../include/mac_b200_chunk.h"

namespace mac_b200 {
namespace {

constexpr int kWarps = 8;

__device__ unsigned g_chunk_status = 0;

// One warp per (row, query head); a lane holds dims [4l, 4l+4).
template <bool kE4m3>
__global__ void __launch_bounds__(kWarps * 32) chunk_rows_kernel(const MacB200ChunkArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (task >= static_cast<int64_t>(a.q_rows) * a.Hq) return;
  const int row = static_cast<int>(task / a.Hq), hq = static_cast<int>(task - static_cast<int64_t>(row) * a.Hq);
  const int kh = hq / (a.Hq / a.Hkv);
  int b = -1;
  for (int i = 0; i < a.B; ++i) {
    const int64_t o0 = a.offsets[i], o1 = a.offsets[i + 1];
    if (o0 < 0 || o1 < o0 || o1 > a.q_rows) {
      if (lane == 0) atomicOr(&g_chunk_status, MAC_B200_STATUS_BAD_REQUEST);
      continue;
    }
    if (row >= o0 && row < o1) b = i;
  }
  if (b < 0) return;
  const int n = a.offsets[b + 1] - a.offsets[b];
  int kv = a.kv_lens[b];
  const int req = a.req_ids[b];
  if (req < 0 || req >= a.req_to_token_rows || kv < 0 || kv > a.req_to_token_stride) {
    if (lane == 0) atomicOr(&g_chunk_status, MAC_B200_STATUS_BAD_REQUEST);
    kv = 0;
  }
  const int64_t p = static_cast<int64_t>(kv) - n + (row - a.offsets[b]);
  int64_t j0 = a.window >= 0 ? p + 1 - a.window : 0;
  if (j0 < 0) j0 = 0;
  const int64_t j1 = kv > 0 ? p + 1 : 0;
  const __nv_bfloat16* qp =
      static_cast<const __nv_bfloat16*>(a.q) + row * a.q_stride0 + hq * 128 + lane * 4;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < 4; ++i) q[i] = __bfloat162float(qp[i]) * a.sm_scale;
  float m = -INFINITY, l = 0.f;
  const int32_t* table = a.req_to_token + static_cast<int64_t>(kv > 0 ? req : 0) * a.req_to_token_stride;
  for (int64_t j = j0; j < j1; ++j) {
    const int64_t tok = table[j];
    float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (tok >= 0 && tok < a.kv_tokens) {
      const int64_t at = tok * a.Hkv + kh;
      if (kE4m3) {
        const uint32_t kc = reinterpret_cast<const uint32_t*>(a.k)[at * 32 + lane];
        const uint32_t vc = reinterpret_cast<const uint32_t*>(a.v)[at * 32 + lane];
        const float ks = kv8_scale(a.k_exp[at]), vs = kv8_scale(a.v_exp[at]);
        for (int i = 0; i < 2; ++i) {
          const float2 kf = kv8_unpack2(kc >> (16 * i)), vf = kv8_unpack2(vc >> (16 * i));
          k[2 * i] = kf.x * ks, k[2 * i + 1] = kf.y * ks;
          v[2 * i] = vf.x * vs, v[2 * i + 1] = vf.y * vs;
        }
      } else {
        const __nv_bfloat16* kp = static_cast<const __nv_bfloat16*>(a.k) + at * 128 + lane * 4;
        const __nv_bfloat16* vp = static_cast<const __nv_bfloat16*>(a.v) + at * 128 + lane * 4;
        for (int i = 0; i < 4; ++i) k[i] = __bfloat162float(kp[i]), v[i] = __bfloat162float(vp[i]);
      }
    } else if (lane == 0) {
      atomicOr(&g_chunk_status, MAC_B200_STATUS_BAD_REQUEST);
    }
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float m2 = fmaxf(m, s);
    const float r = m2 == -INFINITY ? 1.f : __expf(m - m2), w = m2 == -INFINITY ? 0.f : __expf(s - m2);
    m = m2;
    l = l * r + w;
    for (int i = 0; i < 4; ++i) o[i] = o[i] * r + w * v[i];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* op = static_cast<__nv_bfloat16*>(a.out) + (static_cast<int64_t>(row) * a.Hq + hq) * 128 + lane * 4;
  for (int i = 0; i < 4; ++i) op[i] = __float2bfloat16_rn(o[i] * inv);
  if (a.lse && lane == 0) a.lse[static_cast<int64_t>(row) * a.Hq + hq] = l == 0.f ? -INFINITY : m + logf(l);
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int64_t workspace_bytes(int sms) { return static_cast<int64_t>(sms) * 16; }

int chunk_attention(const MacB200ChunkArgs* args, bool e4m3, void* stream_v) {
  MAC_REQUIRE(args != nullptr, "chunk args must not be null");
  const MacB200ChunkArgs& a = *args;
  MAC_REQUIRE(a.D == 128, "chunk attention needs D=128");
  MAC_REQUIRE(a.Hq > 0 && a.Hkv > 0 && a.Hq % a.Hkv == 0 && a.Hq / a.Hkv <= 16,
              "Hq must be Hkv times 1..16");
  MAC_REQUIRE(a.Hkv <= 1024, "Hkv must not exceed 1024");
  MAC_REQUIRE(a.B >= 0 && a.q_rows >= 0, "negative batch");
  MAC_REQUIRE(std::isfinite(a.sm_scale) && a.sm_scale > 0.f, "sm_scale must be positive");
  if (a.B == 0 || a.q_rows == 0) return MAC_B200_OK;
  MAC_REQUIRE(a.q && a.k && a.v && a.req_to_token && a.req_ids && a.offsets && a.kv_lens && a.out && a.workspace,
              "chunk tensors must not be null");
  MAC_REQUIRE(!e4m3 || (a.k_exp && a.v_exp), "the 8-bit pool needs its exponents");
  MAC_REQUIRE(a.kv_tokens > 0 && a.kv_tokens < (int64_t(1) << 31), "the pool must hold 1..2^31-1 rows");
  MAC_REQUIRE(a.req_to_token_rows > 0 && a.req_to_token_stride > 0, "req_to_token must not be empty");
  MAC_REQUIRE(a.q_stride0 >= static_cast<int64_t>(a.Hq) * 128 && a.q_stride0 % 8 == 0,
              "q row stride must be a multiple of 8 and at least Hq*128");
  MAC_REQUIRE(on16(a.q) && on16(a.k) && on16(a.v) && on16(a.out) && on16(a.workspace),
              "chunk tensors must be 16-byte aligned");
  int device = 0;
  MAC_CUDA(cudaGetDevice(&device));
  const int sms = device_sm_count(device);
  MAC_REQUIRE(a.workspace_bytes >= workspace_bytes(sms), "workspace holds %lld bytes, %lld are needed",
              static_cast<long long>(a.workspace_bytes), static_cast<long long>(workspace_bytes(sms)));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const int64_t blocks = (static_cast<int64_t>(a.q_rows) * a.Hq + kWarps - 1) / kWarps;
  MAC_REQUIRE(blocks < (int64_t(1) << 31), "chunk problem too large");
  if (e4m3)
    chunk_rows_kernel<true><<<static_cast<unsigned>(blocks), kWarps * 32, 0, stream>>>(a);
  else
    chunk_rows_kernel<false><<<static_cast<unsigned>(blocks), kWarps * 32, 0, stream>>>(a);
  MAC_CUDA(cudaGetLastError());
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  return MAC_B200_OK;
}

}  // namespace

int take_chunk_status(unsigned* bits) {
  unsigned v = 0;
  MAC_CUDA(cudaMemcpyFromSymbol(&v, g_chunk_status, sizeof(v)));
  if (v != 0) {
    const unsigned zero = 0;
    MAC_CUDA(cudaMemcpyToSymbol(g_chunk_status, &zero, sizeof(zero)));
  }
  *bits = v;
  return MAC_B200_OK;
}

}  // namespace mac_b200

using namespace mac_b200;

extern "C" int mac_b200_chunk_attention_bf16(const MacB200ChunkArgs* args, void* stream) {
  return chunk_attention(args, false, stream);
}

extern "C" int mac_b200_chunk_attention_e4m3(const MacB200ChunkArgs* args, void* stream) {
  return chunk_attention(args, true, stream);
}

extern "C" int mac_b200_chunk_attention_workspace_bytes(int64_t* bytes) {
  MAC_REQUIRE(bytes != nullptr, "bytes must not be null");
  int device = 0;
  MAC_CUDA(cudaGetDevice(&device));
  *bytes = workspace_bytes(device_sm_count(device));
  return MAC_B200_OK;
}
