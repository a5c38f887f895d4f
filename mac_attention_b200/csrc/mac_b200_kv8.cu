// Rows of the 8-bit K/V pool: written (with the decode step's rotation on the way, or without)
// and read back (sm_100a).  Format and rules: include/mac_b200_chunk.h.
//
// Both directions are memory streams: a row of 128 values is 256 bytes in bf16 and 129 held.
// Eight lanes own a row of k and the row of v beside it, 16 values of each: a lane's four 16-byte
// loads are issued before anything is computed (one row at a time: 45 us for the call below), a
// row's maximum is three shuffles away, and the codes leave as one 16-byte store a lane (128 bytes
// a row).  Under the half-split rotation a lane owns dims [8l, 8l+8) and [64+8l, 64+8l+8) instead, so
// both members of a pair are in one thread; its codes leave as two 8-byte stores.  The row's exponent
// is found from the bits of its maximum, no logarithm.
// Measured on a B200 that copies 6564 GB/s: 32768 tokens of 8 heads written in 41 us (0.75 of the copy
// rate, the latency of a block's one round of loads), 100000 read back in 101 us (0.93, memory); one
// to 1000 tokens 4.2 to 4.9 us, the launch.
#include <cuda_bf16.h>

#include "mac_b200_common.h"
#include "mac_b200_kv8.cuh"

#include "../../include/mac_b200_chunk.h"

namespace mac_b200 {
namespace {

constexpr int kKv8Threads = 256;

__device__ unsigned g_kv8_status = 0;

__device__ __forceinline__ int64_t load_loc(const void* p, int is_i64, int64_t n) {
  return is_i64 ? static_cast<const int64_t*>(p)[n]
                : static_cast<int64_t>(static_cast<const int32_t*>(p)[n]);
}
__device__ __forceinline__ void unpack8(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// First dims of a lane's two groups of eight: adjacent, or half a row apart (kSplit).
template <bool kSplit>
__device__ __forceinline__ int dim0(int lane8, int g) {
  return kSplit ? g * 64 + lane8 * 8 : lane8 * 16 + g * 8;
}

template <bool kSplit, bool kVec>
__device__ __forceinline__ void load_row(const __nv_bfloat16* row, int lane8, float (&x)[16]) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const __nv_bfloat16* p = row + dim0<kSplit>(lane8, g);
    if (kVec) {
      unpack8(*reinterpret_cast<const uint4*>(p), x + g * 8);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[g * 8 + i] = __bfloat162float(p[i]);
    }
  }
}

// The eight lanes of a row agree on its exponent and store its codes.
template <bool kSplit>
__device__ __forceinline__ void hold_row(const float (&x)[16], int lane8, uint8_t* codes, uint8_t* exp_byte,
                                         bool write) {
  uint32_t top = 0;                                  // |x| as bits: ordered, NaN above infinity
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (!write) return;
  const bool finite = top < 0x7f800000u;
  const int e = finite ? kv8_exp_of(top) : kKv8NanExp;
  const float inv = finite ? kv8_inverse(e) : 0.f;
  // under the largest scale a code of 256 would stand for 2^128, no bf16 number: 240 at most there
  const float most = e == kKv8MaxExp ? 240.f : 448.f;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fminf(fmaxf(x[4 * i + j] * inv, -most), most);
    w[i] = finite ? kv8_pack4(y[0], y[1], y[2], y[3]) : 0u;
  }
  if (kSplit) {
    *reinterpret_cast<uint2*>(codes + dim0<true>(lane8, 0)) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(codes + dim0<true>(lane8, 1)) = make_uint2(w[2], w[3]);
  } else {
    *reinterpret_cast<uint4*>(codes + lane8 * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lane8 == 0) *exp_byte = static_cast<uint8_t>(e);
}

// Rotates the 16 values that a lane holds of `row`.  Every product and sum is rounded to fp32 by
// itself (no fused multiply-add), so the held row does not depend on how a compiler contracts it.
template <bool kSplit, bool kVec>
__device__ __forceinline__ void rotate_row(const MacB200QuantizeKvArgs& a, const __nv_bfloat16* row,
                                           const float* cs, int lane8, float (&x)[16]) {
  const int half = a.rotary_dim >> 1;
  if (kSplit && kVec) {                              // whole row rotated, pairs (d, d + 64) in the lane
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(cs + lane8 * 8 + i);
      *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(cs + 64 + lane8 * 8 + i);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x0 = x[i], x1 = x[8 + i];
      x[i] = __fsub_rn(__fmul_rn(x0, c[i]), __fmul_rn(x1, s[i]));
      x[8 + i] = __fadd_rn(__fmul_rn(x1, c[i]), __fmul_rn(x0, s[i]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {                     // any rotary_dim, pairing and alignment
    const int d = dim0<kSplit>(lane8, i >> 3) + (i & 7);
    if (d >= a.rotary_dim) continue;
    const int p = a.is_neox ? (d < half ? d : d - half) : d >> 1;
    const bool first = a.is_neox ? d < half : (d & 1) == 0;
    const int d0 = a.is_neox ? p : 2 * p, d1 = a.is_neox ? p + half : 2 * p + 1;
    const float x0 = __bfloat162float(row[d0]), x1 = __bfloat162float(row[d1]);
    const float c = cs[p], s = cs[half + p];
    x[i] = first ? __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s))
                 : __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s));
  }
}

// One task = one KV head of one token, its k row and its v row (four loads a lane before anything is
// computed), or with kRope one query head, after the KV heads.
// kVec: rows are 16-byte aligned (and under kSplit the whole row is rotated in split pairs).
template <bool kRope, bool kSplit, bool kVec>
__global__ void __launch_bounds__(kKv8Threads) kv8_write_kernel(const MacB200QuantizeKvArgs a) {
  const int heads = a.Hkv + (kRope ? a.Hq : 0);
  const int64_t tasks = a.N * heads;
  const int64_t t = (static_cast<int64_t>(blockIdx.x) * kKv8Threads + threadIdx.x) >> 3;
  const int lane8 = threadIdx.x & 7;
  const bool live = t < tasks;                       // whole groups of eight; the shuffles need every lane
  const int64_t n = live ? t / heads : 0;
  int h = live ? static_cast<int>(t - n * heads) : 0;
  const bool is_q = kRope && h >= a.Hkv;
  if (is_q) h -= a.Hkv;
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(is_q ? a.q : a.k) +
                             n * (is_q ? a.q_stride0 : a.k_stride0) + static_cast<int64_t>(h) * 128;
  float x[16] = {}, y[16] = {};
  int64_t loc = -1, pos = 0;
  if (live) {
    load_row<kSplit, kVec>(row, lane8, x);
    if (!is_q) {
      load_row<kSplit, kVec>(static_cast<const __nv_bfloat16*>(a.v) + n * a.v_stride0 + static_cast<int64_t>(h) * 128,
                             lane8, y);
      loc = load_loc(a.cache_locs, a.cache_locs_i64, n);
    }
    if (kRope) pos = load_loc(a.positions, a.positions_i64, n);
  }
  bool ok = live;
  if (kRope && live) {
    ok = pos >= 0 && pos < a.max_positions;
    if (!ok && lane8 == 0) atomicOr(&g_kv8_status, MAC_B200_STATUS_BAD_REQUEST);
    if (ok) rotate_row<kSplit, kVec>(a, row, a.cos_sin_cache + pos * a.cos_sin_stride0, lane8, x);
  }
  if (is_q && ok) {
    __nv_bfloat16* post = static_cast<__nv_bfloat16*>(a.q_post) + (n * a.Hq + h) * 128;
#pragma unroll
    for (int g = 0; g < 2; ++g)
      *reinterpret_cast<uint4*>(post + dim0<kSplit>(lane8, g)) =
          make_uint4(pack_bf16(x[g * 8], x[g * 8 + 1]), pack_bf16(x[g * 8 + 2], x[g * 8 + 3]),
                     pack_bf16(x[g * 8 + 4], x[g * 8 + 5]), pack_bf16(x[g * 8 + 6], x[g * 8 + 7]));
  }
  const bool write = ok && !is_q && loc >= 0 && loc < a.kv_pool_tokens;
  const int64_t at = (write ? loc : 0) * a.Hkv + (write ? h : 0);
  hold_row<kSplit>(x, lane8, static_cast<uint8_t*>(a.k_pool) + at * 128, a.k_exp + at, write);
  hold_row<kSplit>(y, lane8, static_cast<uint8_t*>(a.v_pool) + at * 128, a.v_exp + at, write);
}

// One task = one (row, K or V, head): 16 codes a lane in one load, 16 bf16 out.
__global__ void __launch_bounds__(kKv8Threads) kv8_read_kernel(const MacB200DequantizeKvArgs a) {
  const int64_t t = (static_cast<int64_t>(blockIdx.x) * kKv8Threads + threadIdx.x) >> 3;
  const int lane8 = threadIdx.x & 7;
  const int64_t n = t / a.Hkv;
  if (n >= a.N) return;
  const int h = static_cast<int>(t - n * a.Hkv);
  const int64_t from = load_loc(a.src_locs, a.src_locs_i64, n);
  const int64_t to = a.dst_locs ? load_loc(a.dst_locs, a.dst_locs_i64, n) : n;
  if (from < 0 || from >= a.src_tokens || to < 0 || to >= a.dst_tokens) return;
  const int64_t src = from * a.Hkv + h, dst = to * a.Hkv + h;
  const uint4 kc = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.k_pool) + src * 128 + lane8 * 16);
  const uint4 vc = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.v_pool) + src * 128 + lane8 * 16);
  const float ks = kv8_scale(a.k_exp[src]), vs = kv8_scale(a.v_exp[src]);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint4 c4 = which ? vc : kc;
    const float s = which ? vs : ks;
    const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = kv8_unpack2(c[i >> 1] >> ((i & 1) * 16));
      w[i] = pack_bf16(f.x * s, f.y * s);
    }
    uint4* o = reinterpret_cast<uint4*>(static_cast<char*>(which ? a.v_buffer : a.k_buffer) + dst * 256 + lane8 * 32);
    store32(o, w, (reinterpret_cast<uintptr_t>(o) & 31u) == 0u);
  }
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// blocks of a launch with eight lanes a task, or 0 when there are too many
unsigned blocks_for(int64_t tasks) {
  constexpr int64_t per = kKv8Threads / 8;
  const int64_t blocks = (tasks + per - 1) / per;
  return blocks < (int64_t(1) << 31) ? static_cast<unsigned>(blocks) : 0u;
}

}  // namespace

int kv8_status_word(unsigned** word) {
  MAC_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(word), g_kv8_status));
  return MAC_B200_OK;
}

}  // namespace mac_b200

using namespace mac_b200;

extern "C" int mac_b200_quantize_kv_e4m3(const MacB200QuantizeKvArgs* args, void* stream_v) {
  MAC_REQUIRE(args != nullptr, "quantize args must not be null");
  const MacB200QuantizeKvArgs& a = *args;
  MAC_REQUIRE(a.D == 128, "the 8-bit pool needs D=128");
  MAC_REQUIRE(a.N >= 0, "negative batch");
  MAC_REQUIRE(a.Hkv > 0 && a.Hkv <= 65536, "invalid Hkv");
  MAC_REQUIRE(a.kv_pool_tokens >= 0, "negative pool size");
  const bool rope = a.q != nullptr;
  if (a.N == 0) return MAC_B200_OK;
  MAC_REQUIRE(a.N <= (int64_t(1) << 31), "too many tokens");
  MAC_REQUIRE(a.k && a.v && a.k_pool && a.v_pool && a.k_exp && a.v_exp && a.cache_locs,
              "quantize tensors must not be null");
  MAC_REQUIRE(on16(a.k_pool) && on16(a.v_pool), "the pool must be 16-byte aligned");
  MAC_REQUIRE(!rope || (a.q_post && a.cos_sin_cache && a.positions), "rope tensors must not be null");
  MAC_REQUIRE(!rope || (a.Hq > 0 && a.Hq <= 65536), "invalid Hq");
  MAC_REQUIRE(!rope || (a.rotary_dim > 0 && a.rotary_dim <= 128 && a.rotary_dim % 2 == 0),
              "invalid rotary_dim");
  MAC_REQUIRE(!rope || on16(a.q_post), "q_post must be 16-byte aligned");
  if (rope) {                                        // rows are read by other threads than those that write them
    const int64_t last = a.N - 1, post_bytes = a.N * a.Hq * 256;
    MAC_REQUIRE(!byte_ranges_meet(a.q, (last * a.q_stride0 + a.Hq * int64_t{128}) * 2, a.q_post, post_bytes) &&
                    !byte_ranges_meet(a.k, (last * a.k_stride0 + a.Hkv * int64_t{128}) * 2, a.q_post, post_bytes) &&
                    !byte_ranges_meet(a.v, (last * a.v_stride0 + a.Hkv * int64_t{128}) * 2, a.q_post, post_bytes),
                "q_post must not share memory with q, k or v");
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const int64_t heads = static_cast<int64_t>(a.Hkv) + (rope ? a.Hq : 0);
  const unsigned blocks = blocks_for(a.N * heads);
  MAC_REQUIRE(blocks > 0, "quantize problem too large");
  const bool vec = on16(a.k) && on16(a.v) && a.k_stride0 % 8 == 0 && a.v_stride0 % 8 == 0;
  if (!rope) {
    if (vec)
      kv8_write_kernel<false, false, true><<<blocks, kKv8Threads, 0, stream>>>(a);
    else
      kv8_write_kernel<false, false, false><<<blocks, kKv8Threads, 0, stream>>>(a);
  } else {
    const bool split = vec && on16(a.q) && a.q_stride0 % 8 == 0 && on16(a.cos_sin_cache) &&
                       a.cos_sin_stride0 % 4 == 0 && a.is_neox && a.rotary_dim == 128;
    if (split)
      kv8_write_kernel<true, true, true><<<blocks, kKv8Threads, 0, stream>>>(a);
    else
      kv8_write_kernel<true, false, false><<<blocks, kKv8Threads, 0, stream>>>(a);
  }
  MAC_CUDA(cudaGetLastError());
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  return MAC_B200_OK;
}

extern "C" int mac_b200_dequantize_kv_e4m3(const MacB200DequantizeKvArgs* args, void* stream_v) {
  MAC_REQUIRE(args != nullptr, "dequantize args must not be null");
  const MacB200DequantizeKvArgs& a = *args;
  MAC_REQUIRE(a.D == 128, "the 8-bit pool needs D=128");
  MAC_REQUIRE(a.N >= 0, "negative row count");
  MAC_REQUIRE(a.Hkv > 0 && a.Hkv <= 65536, "invalid Hkv");
  MAC_REQUIRE(a.src_tokens >= 0 && a.dst_tokens >= 0, "negative pool size");
  if (a.N == 0 || a.src_tokens == 0 || a.dst_tokens == 0) return MAC_B200_OK;
  MAC_REQUIRE(a.N <= (int64_t(1) << 31), "too many rows");
  MAC_REQUIRE(a.k_pool && a.v_pool && a.k_exp && a.v_exp && a.src_locs && a.k_buffer && a.v_buffer,
              "dequantize tensors must not be null");
  MAC_REQUIRE(on16(a.k_pool) && on16(a.v_pool) && on16(a.k_buffer) && on16(a.v_buffer),
              "the pools must be 16-byte aligned");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const unsigned blocks = blocks_for(a.N * a.Hkv);
  MAC_REQUIRE(blocks > 0, "dequantize problem too large");
  kv8_read_kernel<<<blocks, kKv8Threads, 0, stream>>>(a);
  MAC_CUDA(cudaGetLastError());
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  return MAC_B200_OK;
}
