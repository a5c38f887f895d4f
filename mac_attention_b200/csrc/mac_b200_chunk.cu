// Attention of a chunk of new tokens over the paged K/V pool, bf16 or e4m3 (sm_100a).
// Semantics: include/mac_b200_chunk.h.
//
// Rows.  A KV head's G query heads see the same keys, so the rows of a tile are (token, query
// head) pairs: 128/G tokens x G heads fill the 128 rows of a tcgen05 product.  A UNIT of work is
// (request, KV head, one or two tiles of rows) with the keys that its rows attend together, in
// blocks of 128 keys.  Two tiles ("dual") share every staged K/V block, which halves the traffic
// through shared memory; in a unit of one tile ("single": decode, drafted tokens, a prompt's
// remainder, and every unit of a call with too few tiles to fill the GPU with pairs) the two
// softmax streams take alternate blocks of the same rows, and their results are joined in place:
// both streams' accumulators of a row lie in the same lane of tensor memory.  Either way two
// streams are in flight, and while one is in its softmax the other's products run.
//
// Split.  All blocks of all units lie on one line (request, KV head, tile, block) that is cut into
// equal parts, one per CTA: no tail wave whatever the lengths.  Every CTA works its part out from
// the lengths by itself; no CTA waits for another.  A unit that a cut falls into leaves
// unnormalised fp32 results in the workspace, and a second small kernel joins them in the order of
// the parts, so the result does not depend on timing.
//
// Roles of a CTA (one per SM):
//   the last eight   softmax streams 0 and 1, a thread a row: scores from tensor memory, running
//                    maximum and sum in fp32, bf16 weights back over the scores, results out
//   warps 0, 1       issue the streams' products: S = Q K^T from shared memory, O += P V with P from
//                    tensor memory and V from the rows as they lie in the pool (keys x dims); products
//                    that differ in shape are not promised to run in the order of issue, so where one
//                    writes what another reads it is issued after that one is done
//   warps 4-7 (-15)  fetch K/V rows by the page table into the swizzled operand layout (cp.async; the
//                    8-bit pool's rows by way of a raw buffer, widened to bf16)
//   warp 2           works out the units of this CTA's part, fetches the query tiles
// A stream goes in steps of 64 keys with two score buffers, so the products of the next step run
// while a step is in its softmax (steps of 128 keys leave room for one buffer a stream).
// The running maximum is kept until a row's scores exceed it by 2^8 in weight: the rescaling of O
// is rare, and exact when it happens.  Weights are rounded to bf16 for the second product (the
// operand type); the sum of weights is taken before that rounding, in fp32.
//
// Measured (B200: 6564 GB/s copied, 1675 TFLOP/s of a bf16 product; calls on inputs that change from call
// to call, here and below, unless it says otherwise):
//   decode, 16 requests x 30000-32768 tokens, 32 / 8 heads: 392-399 us, 0.80 of the copy rate (the same
//     call over and over 338, 0.94); the 8-bit pool 389-398 us, 0.40 (353-370, 0.44): no one part bounds
//     it (without the widening's stores 0.92 of the time, without the row fetches 0.96, without the
//     softmax 0.93), the chain through the ring's few positions does
//   prompt, 4096 tokens behind 28672 cached, 32 / 8 heads: 2285-2319 us, 889-902 TFLOP/s; 2 x 1024 tokens
//     of 8192 over the 8-bit pool 545-554 us, 841-854 TFLOP/s.  Without the softmax's arithmetic such a call
//     still takes 0.85 of its time: a product of 128 x 64 from shared memory is bound by the reads
//     of its operands (412 cycles for 256 of arithmetic) and the hand-overs between the products
//     and the softmax are not hidden entirely.  ncu (1024 tokens of 8192, 64 / 8 heads): tensor cores
//     46 %, issue slots 45 %, exponentials 46 % of the cycles.
//   8 prompts of 1500-2048 in a band of 1024: 564-573 us, 634-645 TFLOP/s (masked halves of blocks count
//     as none)
//   three requests of drafted tokens behind 1000: 22 us a call by itself; a single token of 128, calls in
//     a row within one graph, 11.4 us, of which 3 are set-up (lengths, tensor memory) and 5 the chain of
//     one block's steps
// No gain, measured on the same calls: steps of 128 keys, one warp that issues for both streams,
// turns between the streams' products, two threads a row, a quarter of the exponentials by a
// polynomial, bulk row gathers instead of cp.async (80 cycles each to issue).
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "mac_b200_chunk_ring.h"
#include "mac_b200_common.h"
#include "mac_b200_kv8.cuh"

#include "../../include/mac_b200_chunk.h"

namespace mac_b200 {
namespace {

constexpr int kBlk = 128;                  // keys of a block
constexpr int kRows = 128;                 // rows of a tile
constexpr int kHalf = 64;                  // keys of a step: what a stream takes from scores to weights at once
constexpr int kHalfBytes = 128 * 128;      // 128 rows x 64 bf16 in the 128-byte-swizzled layout
constexpr int kTileBytes = 2 * kHalfBytes;
constexpr int kMaxStages = 5;              // K/V blocks in shared memory
constexpr int kItems = 4;                  // units announced ahead
// Warps by role.  The issuing warps come first: a scheduler prefers its older warps.
constexpr int kMmaWarp = 0, kPlanWarp = 2, kLoadWarp = 4, kSoftmaxWarps = 8;
constexpr int kUnitCells = 1;              // what a unit costs beside its blocks, in blocks
constexpr int kMinCells = 2;               // least work worth a CTA of its own (1, 4, 6: up to 5 us slower)
constexpr int kJoinRows = 16;              // rows of a unit that a block of the second kernel joins
constexpr int kTmemCols = 512;             // S0 S1 O0 O1; the weights lie over the scores
constexpr long long kWaitLimitClocks = 4000000000ll;   // about two seconds

// The workspace: a list of the units that were cut (entry c: the one that begins in CTA c's part
// and ends behind it), then two slots a CTA for a part's unnormalised results, 256 rows each.
struct Cut {
  int parts, kh, tok0, ntok;
};
constexpr int kMaxCtas = 1024;
constexpr int64_t kCutBytes = kMaxCtas * static_cast<int64_t>(sizeof(Cut));
constexpr int kSlotRows = 2 * kRows;
constexpr int64_t kSlotFloats = kSlotRows * 128;       // [four dims][row]: a warp stores whole lines
constexpr int64_t kSlotBytes = kSlotFloats * 4 + kSlotRows * 8;   // then (maximum, sum) of each row

// bf16 x bf16 -> fp32, M 128: N 64 keys of the first product; N 128 dims of the second, whose B
// operand is dim-contiguous
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
constexpr uint32_t kIdescQk = kIdesc | ((64u >> 3) << 17);
constexpr uint32_t kIdescPv = kIdesc | ((128u >> 3) << 17) | (1u << 16);

__device__ unsigned g_chunk_status = 0;

struct Item {
  int valid, dual;
  int kh, req;             // KV head, row of the page table
  int tok0, ntok;          // first row of q, tokens
  int pos0;                // position of the first token (negative: attends nothing)
  int k0, khi;             // keys [k0, khi) are attended by some row of the unit
  int blk0, nblk;          // this part's blocks, counted from k0
  int qbuf;                // query buffer of a single unit
  int parts;               // CTAs that share the unit
  int slot;
  unsigned nonfinite;      // a value that only some rows attend was infinite or NaN
};

struct Control {
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages];
  uint64_t q_full[2], q_empty[2], s_full[2][2], p_full[2][2], o_done[2][2];
  uint64_t item_full[kItems], item_empty[kItems], join;
  Item items[kItems];
  long long scan[24];      // a word a warp
  long long start_pos;     // where request start_b begins on the line
  int start_b;
  uint32_t tmem;
  unsigned abort;
  float2 ml[2][kRows];     // a single unit's maxima and sums, by stream
};

// Shared memory: two query tiles, the ring of K/V blocks (the 8-bit pool's with the second tile where it is
// not needed), for the 8-bit pool the raw rows on their way (each thread of the loading warps reads back
// what it fetched itself), the control words.
// Registers a thread after the warpgroups have traded theirs:
//   bf16: 128 * 64 + 128 * 160 + 256 * 144 = 512 * 128,  e4m3: 128 * 64 + 384 * 48 + 256 * 128 <= 768 * 80
constexpr int kSmemQ = 0;
constexpr int kSmemKv = 2 * kTileBytes;
template <bool kE4m3>
struct Layout {
  static constexpr int kLoadWarps = 4 * RingShape<kE4m3>::kGroups;
  static constexpr int kWarpRows = 32;                   // rows of a block that a loading warp fetches
  static constexpr int kSoftmaxWarp = kLoadWarp + kLoadWarps;
  static constexpr int kThreads = 32 * (kSoftmaxWarp + kSoftmaxWarps);
  static constexpr int kLaunchRegs = kE4m3 ? 80 : 128, kControlRegs = 64;
  static constexpr int kLoadRegs = kE4m3 ? 48 : 160, kSoftmaxRegs = kE4m3 ? 128 : 144;
  static constexpr int kStages = RingShape<kE4m3>::kStages;
  static constexpr int kRawRows = kWarpRows * 128;       // of a warp and a ring position
  // with the 16 bytes around each row's exponent, and the table's entries of three positions later
  static constexpr int kRawExps = kRawRows, kRawEntries = kRawExps + kWarpRows * 16;
  static constexpr int kRawBytes = kRawEntries + kWarpRows * 4;
  static constexpr int kRaw = kSmemKv + kStages * kTileBytes;
  static constexpr int kControl = kRaw + (kE4m3 ? kLoadWarps * kRawBytes : 0);
  static constexpr int kBytes = kControl + static_cast<int>(sizeof(Control));
};
template <typename L>
constexpr bool registers_suffice() {
  return 128 * L::kControlRegs + 32 * L::kLoadWarps * L::kLoadRegs + 32 * kSoftmaxWarps * L::kSoftmaxRegs <=
         L::kThreads * L::kLaunchRegs;
}
static_assert(registers_suffice<Layout<false>>() && registers_suffice<Layout<true>>(),
              "warps that ask for more registers than the CTA was launched with wait for ever");
static_assert(Layout<false>::kBytes <= 232448 && Layout<true>::kBytes <= 232448, "shared memory of a CTA");

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for the phase of the given parity.  False when the limit ran out here or in another warp of
// the CTA: the caller leaves its loop.  For one lane by itself, or where a vote follows.  Short on
// purpose: it stands at two dozen places, and what the warps of a scheduler execute in turn has to stay
// in its instruction cache.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, unsigned* abort_flag) {
  const uint32_t b = smem_u32(bar);
  if (mbar_try(b, parity & 1u)) return true;
  const long long t0 = clock64();
  while (!mbar_try(b, parity & 1u)) {                    // each try may itself block for a while
    if (*reinterpret_cast<volatile unsigned*>(abort_flag) != 0u) return false;
    if (clock64() - t0 > kWaitLimitClocks) {
      *reinterpret_cast<volatile unsigned*>(abort_flag) = MAC_B200_STATUS_COPY_TIMEOUT;   // reported at the end
      return false;
    }
  }
  return true;
}
// The same for a warp whose lanes go on together.  The limit can run out for one lane and not for the
// next; lanes that then took different ways would meet each other's votes, and wait for ever.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Operand in shared memory, 128-byte swizzle, eight-row groups 1024 bytes apart.  `lead`: bytes
// between the two 64-dim halves when the operand is dim-contiguous (unused when key-contiguous).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(2) << 61);
}
// D (+)= A B^T, 128 x 64 x 16: A and B from shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(kIdescQk), "r"(accumulate)
      : "memory");
}
// D (+)= A B, 128 x 128 x 16: A from tensor memory, B dim-contiguous from shared memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(kIdescPv), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
// 32 consecutive columns of this thread's tensor-memory lane; tmem_ld_wait() before they are used
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// ties loaded registers to the wait before it: nothing that uses them may move above it
__device__ __forceinline__ void loaded(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// the largest of three, NaN if any is NaN
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// a load that stays where it is written: ahead of its use
__device__ __forceinline__ int load_early(const int32_t* p) {
  int v;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
// 16 bytes, or 16 zeros when `bytes` is 0
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// arrives on `bar` once this thread's copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// rows written by cp.async (or by stores) that a barrier has made visible here, to the copy
// engine's and the tensor cores' view of shared memory
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// a value that every lane holds alike, so that the compiler knows it
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// ---------------------------------------------------------------------------- units on the line
struct Request {
  int row0, n, kv, req;
};
// `report`: set the status bit for what cannot be run (one thread of the grid does)
__device__ __forceinline__ Request load_request(const MacB200ChunkArgs& a, int b, bool report) {
  Request r;
  const int o0 = a.offsets[b], o1 = a.offsets[b + 1];
  r.row0 = o0;
  r.n = o1 - o0;
  r.req = a.req_ids[b];
  r.kv = a.kv_lens[b];
  bool bad = false;
  if (o0 < 0 || o1 < o0 || o1 > a.q_rows) {
    r.n = 0;
    bad = true;
  } else if (r.req < 0 || r.req >= a.req_to_token_rows || r.kv < 0 || r.kv > a.req_to_token_stride) {
    r.kv = 0;                                            // rows without keys
    r.req = 0;
    bad = true;
  }
  if (bad && report) atomicOr(&g_chunk_status, MAC_B200_STATUS_BAD_REQUEST);
  return r;
}
struct Unit {
  int t0, ntok;            // tokens of the request
  int k0, khi, nblk;
};
// `span`: tokens of a whole unit (one or two tiles)
__device__ __forceinline__ Unit unit_of(const Request& r, int window, int span, int t) {
  Unit u;
  u.t0 = t * span;
  u.ntok = min(span, r.n - u.t0);
  const int p0 = r.kv - r.n + u.t0;
  u.khi = max(0, p0 + u.ntok);
  u.k0 = 0;
  if (window >= 0) u.k0 = static_cast<int>(max(0ll, static_cast<long long>(p0) + 1 - window));
  u.nblk = window == 0 || u.k0 >= u.khi ? 0 : (u.khi - u.k0 + kBlk - 1) / kBlk;
  return u;
}
// Cells of a unit on the line: what it costs beside its blocks, then its blocks.
__device__ __forceinline__ int cells_of(const Unit& u) { return kUnitCells + u.nblk; }
__device__ __forceinline__ long long head_cells(const Request& r, int window, int span) {
  long long c = 0;
  for (int t = 0; t * span < r.n; ++t) c += cells_of(unit_of(r, window, span, t));
  return c;
}

// Sum over the CTA of `mine`; `before` gets what the threads before this one hold.
template <int kThreads>
__device__ __forceinline__ long long scan_cta(long long mine, long long& before, long long* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  long long total = 0;
  before = x - mine;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warps[w];
    total += warps[w];
  }
  return total;
}

// The ring holds K and V in turn when both streams use each block, and is one K ahead when the
// streams alternate (K0 K1 V0 K2 V1 ...).  Where in a unit's positions block `blk`'s V is:
__device__ __forceinline__ int ring_v(int dual, int blk, int nblk) {
  return dual ? 2 * blk + 1 : min(2 * blk + 2, 2 * nblk - 1);
}

// Dims [d, d + 2) of the value of key `key`; zeros where the page table leads outside the pool.
template <bool kE4m3>
__device__ __forceinline__ float2 value_pair(const MacB200ChunkArgs& a, const Item& it, int key, int d) {
  const int tok = a.req_to_token[static_cast<int64_t>(it.req) * a.req_to_token_stride + key];
  if (tok < 0 || tok >= a.kv_tokens) return make_float2(0.f, 0.f);
  const int64_t row = static_cast<int64_t>(tok) * a.Hkv + it.kh;
  if (!kE4m3) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const char*>(a.v) + row * 256 + d * 2);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  const float2 x = kv8_unpack2(*reinterpret_cast<const uint16_t*>(static_cast<const char*>(a.v) + row * 128 + d));
  const uint32_t w = pack_bf16(x.x * kv8_scale(a.v_exp[row]), x.y * kv8_scale(a.v_exp[row]));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// ------------------------------------------------------------------- rows of the 8-bit pool
__device__ __forceinline__ uint32_t mul_bf16(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
// A row's scale as a pair of bf16: 2^(e-127), NaN for e = 255.
__device__ __forceinline__ uint32_t scale_pair(int e) {
  const uint32_t f = e == kKv8NanExp ? 0x7fc0u : e == 0 ? 0x0040u : static_cast<uint32_t>(e) << 7;
  return f | (f << 16);
}
// Eight codes of a row to bf16 (four words): through fp16 and fp32, which hold every code, to bf16,
// which does too, and then the scale, a power of two.  (200 cycles a warp for 64 codes a lane;
// moving the bits by hand took 290 and a check for codes of NaN beside it.)
__device__ __forceinline__ uint4 widen8(const uint2& codes, uint32_t scale) {
  const uint32_t c[2] = {codes.x, codes.y};
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = kv8_unpack2(c[i >> 1] >> ((i & 1) * 16));
    w[i] = mul_bf16(pack_bf16(x.x, x.y), scale);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool kE4m3>
__global__ void __launch_bounds__(Layout<kE4m3>::kThreads, 1)
chunk_attention_kernel(const MacB200ChunkArgs a, const __grid_constant__ CUtensorMap q_map) {
  extern __shared__ __align__(1024) uint8_t smem[];      // the swizzle repeats every 1024 bytes
  // the joining kernel may be set up from here on; it waits for this one's end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using L = Layout<kE4m3>;
  constexpr int kGroups = RingShape<kE4m3>::kGroups;     // of loading warps, that take positions in turn
  constexpr int kStages = L::kStages, kThreads = L::kThreads, kLoadWarps = L::kLoadWarps;
  constexpr int kSoftmaxWarp = L::kSoftmaxWarp;
  Control& ctl = *reinterpret_cast<Control*>(smem + Layout<kE4m3>::kControl);
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const int G = a.Hq / a.Hkv;
  const int tile_tokens = kRows / G;
  Cut* const cuts = static_cast<Cut*>(a.workspace);

  // ---- the line: this CTA's part of it, and the request that the part begins in
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  long long mine = 0, before;
  const Request mine0 = b0 < b1 ? load_request(a, b0, blockIdx.x == 0) : Request{};   // most calls: a thread's only one
  for (int b = b0; b < b1; ++b)
    mine += a.Hkv * static_cast<long long>(
                        ((b == b0 ? mine0 : load_request(a, b, blockIdx.x == 0)).n + tile_tokens - 1) / tile_tokens);
  // pairs of tiles once there are enough of them for every CTA
  const int span = scan_cta<kThreads>(mine, before, ctl.scan) >= 2ll * gridDim.x ? 2 * tile_tokens : tile_tokens;
  // The 8-bit pool's ring is short: three positions.  Where every unit is of one tile the second query
  // buffer, in front of it, joins it as a fourth (decode 390 us, 405 with three; a sixth position of
  // bf16 gains nothing).  Four are no multiple of the three groups that fill them: see wait_to_fill().
  const int stages = span == tile_tokens ? kStages + RingShape<kE4m3>::kSpare : kStages;
  uint8_t* const ring = smem + kSmemKv - (stages - kStages) * kTileBytes;
  long long units = 0;
  mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Request r = b == b0 ? mine0 : load_request(a, b, false);
    mine += a.Hkv * head_cells(r, a.window, span);
    units += a.Hkv * static_cast<long long>((r.n + span - 1) / span);
  }
  long long unused;
  units = scan_cta<kThreads>(units, unused, ctl.scan);
  const long long total = scan_cta<kThreads>(mine, before, ctl.scan);
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), max(units, total / kMinCells)));
  if (tid == 0) cuts[blockIdx.x].parts = 0;
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  if ((smem_u32(smem) & 1023u) != 0u) {                  // the operand layout would not hold
    if (tid == 0) atomicOr(&g_chunk_status, MAC_B200_STATUS_SCHED_OVERFLOW);
    return;
  }
  const long long lo = total * blockIdx.x / ctas, hi = total * (blockIdx.x + 1) / ctas;
  if (lo >= before && lo < before + mine) {
    long long at = before;
    for (int b = b0; b < b1; ++b) {
      const long long len = a.Hkv * head_cells(b == b0 ? mine0 : load_request(a, b, false), a.window, span);
      if (lo < at + len) {
        ctl.start_b = b;
        ctl.start_pos = at;
        break;
      }
      at += len;
    }
  }

  // ---- barriers, tensor memory
  if (tid == 0) {
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(&ctl.kv_full[i], kE4m3 ? 4 : kLoadWarps * 32);
      mbar_init(&ctl.kv_empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.q_full[i], 1);
      mbar_init(&ctl.q_empty[i], 2);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&ctl.s_full[i][h], 1);
        mbar_init(&ctl.p_full[i][h], kSoftmaxWarps / 2);
        mbar_init(&ctl.o_done[i][h], 1);
      }
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&ctl.item_full[i], 1);
      mbar_init(&ctl.item_empty[i], kSoftmaxWarps + kLoadWarps + 2);
    }
    mbar_init(&ctl.join, kSoftmaxWarps);
    ctl.abort = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(ctl.tmem)));
  unsigned* const abort_flag = &ctl.abort;

  if (warp >= kLoadWarp && warp < kSoftmaxWarp) {
    if constexpr (kE4m3)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kLoadRegs));
    else
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kLoadRegs));
    const int part = ((warp - kLoadWarp) & 3) * L::kWarpRows;   // this warp's rows of a block
    const int group = (warp - kLoadWarp) >> 2;           // e4m3: of four warps, for every third position
    uint32_t st = 0, phase = 1;                          // of the ring position to fill next
    int own = group;                                     // e4m3: the group's next position of the unit
    if (kE4m3) st = group;
    bool ok = true;
    // bf16: sixteen lanes a row, straight into the swizzled operand layout (cp.async).
    // e4m3: eight lanes a row, into a raw buffer ahead of time (48 KB of them; held in registers the rows
    // were waited for all at once), then widened to bf16 with their scales on the way into the operand
    // layout.  The widened rows are exact: from there on the two pools go the same way.  Four warps
    // take every third position, so three are widened at once (eight warps on one after the other: 8 %
    // more for the decode call above).
    constexpr int kLanes = kE4m3 ? 8 : 16;               // of a row
    const int sub = lane / kLanes, c = lane % kLanes;    // row of a load, 16 bytes of it
    const int64_t row_stride = static_cast<int64_t>(a.Hkv) * (kE4m3 ? 128 : 256);
    uint32_t to[4];                                      // bf16: where this lane's chunk goes in rows 2i + sub
    if constexpr (!kE4m3) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = part + 2 * i + sub;
        to[i] = smem_u32(ring) + (c >> 3) * kHalfBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
      }
    }
    uint8_t* const wide = ring + (c >> 2) * kHalfBytes + (part + sub) * 128;   // e4m3: the same, widened
    uint8_t* const raw = smem + L::kRaw + (warp - kLoadWarp) * L::kRawBytes;
    for (int it = 0; ok; ++it) {
      const int slot = it & (kItems - 1);
      ok = warp_wait(&ctl.item_full[slot], it / kItems, abort_flag);
      if (!ok) break;
      const Item& o = ctl.items[slot];
      if (!o.valid) break;
      const int dual = o.dual, nblk = o.nblk, khi = o.khi, kh = o.kh;
      const int first = o.k0 + o.blk0 * kBlk;
      const int64_t col = kh * (kE4m3 ? 128 : 256) + c * 16;
      const int32_t* table = a.req_to_token + static_cast<int64_t>(o.req) * a.req_to_token_stride;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.item_empty[slot]);
      const int n = 2 * nblk;
      if constexpr (!kE4m3) {
        // Key `lane` of this warp's part of the next ring position: the key, and what the table says of
        // it.  Table entries are asked for ahead and looked at when they are needed.
        struct Entry {
          int key, row;
          bool is_v;
        };
        int k_next = 0, v_next = 0;                        // blocks asked for; see ring_v()
        auto entry_of = [&]() {
          Entry e{khi, 0, false};
          if (v_next == nblk) return e;
          e.is_v = k_next == nblk || k_next > v_next + (dual ? 0 : 1);
          e.key = first + (e.is_v ? v_next++ : k_next++) * kBlk + part + lane;
          if (e.key < khi) e.row = load_early(table + e.key);
          return e;
        };
        // the pool row; -1: no key, or one outside the pool (reported): arrives as zeros
        auto row_of = [&](const Entry& e) {
          if (e.key >= khi) return -1;
          if (e.row >= 0 && e.row < a.kv_tokens) return e.row;
          atomicOr(&g_chunk_status, MAC_B200_STATUS_BAD_REQUEST);
          return -1;
        };
        // Entries are refilled where they were used: moved on to another one they would be waited for.
        Entry e[2] = {entry_of(), entry_of()};
        for (int i0 = 0; i0 < n && ok; i0 += 2) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {                  // n is even
            ok = warp_wait(&ctl.kv_empty[st], phase, abort_flag);
            if (!ok) break;
            const char* src = static_cast<const char*>(e[i].is_v ? a.v : a.k) + col;
            const int row = row_of(e[i]);
            e[i] = entry_of();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int tok = __shfl_sync(0xffffffffu, row, 2 * j + sub);
              cp_async16(to[j & 3] + (j >> 2) * 1024 + st * kTileBytes, src + (tok < 0 ? 0 : tok) * row_stride,
                         tok < 0 ? 0 : 16);
            }
            cp_async_arrive(&ctl.kv_full[st]);
            if (++st == stages) st = 0, phase ^= 1u;
          }
        }
      } else {
        // This group's positions of the unit are i0, i0 + 3, ...
        const int i0 = own;
        // the key of this lane's row in position i of the unit (see ring_v()); khi: none
        auto key_of = [&](int i, bool& is_v) {
          is_v = dual ? (i & 1) != 0 : i == n - 1 || (i > 0 && (i & 1) == 0);
          const int blk = dual ? i >> 1 : is_v ? (i == n - 1 ? nblk : i >> 1) - 1 : (i + 1) >> 1;
          return i < n ? first + blk * kBlk + part + lane : khi;
        };
        auto ask = [&](int i) {
          bool is_v;
          const int key = key_of(i, is_v);
          if (key < khi) cp_async4(smem_u32(raw + L::kRawEntries + lane * 4), table + key, 4);
        };
        int row = 0, bytes = 0;                          // of a position: this lane's pool row, its exponent's place
        bool is_v = false;
        auto asked = [&](int i) {
          const int key = key_of(i, is_v);
          row = -1;
          if (key < khi) {
            row = *reinterpret_cast<const int*>(raw + L::kRawEntries + lane * 4);
            if (row < 0 || row >= a.kv_tokens) {
              row = -1;
              atomicOr(&g_chunk_status, MAC_B200_STATUS_BAD_REQUEST);
            }
          }
        };
        auto fetch_exps = [&]() {
          const uint8_t* exps = (is_v ? a.v_exp : a.k_exp) + static_cast<int64_t>(max(row, 0)) * a.Hkv + kh;
          bytes = static_cast<int>(reinterpret_cast<uintptr_t>(exps) & 15u);
          const uint8_t* const end = (is_v ? a.v_exp : a.k_exp) + a.kv_tokens * a.Hkv;
          // 16-byte copies pass the L1 cache by; single words would each hold a line of the little that
          // this much shared memory leaves of it, and wait for one
          cp_async16(smem_u32(raw + L::kRawExps + lane * 16), exps - bytes,
                     row < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(16), end - (exps - bytes))));
        };
        auto fetch_half = [&](int half) {
          const uint8_t* src = static_cast<const uint8_t*>(is_v ? a.v : a.k) + col;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int tok = __shfl_sync(0xffffffffu, row, half * 16 + 4 * j + sub);
            cp_async16(smem_u32(raw + half * 2048 + j * 512 + lane * 16), src + max(tok, 0) * row_stride,
                       tok < 0 ? 0 : 16);
          }
        };
        // Lanes of a row's second half widen and store their two chunks in the other order: no two lanes
        // of a row store to the same bank.
        const int flip = c >= 4 ? 1 : 0;
        const int c0 = 2 * (c & 3) + flip;
        auto store_half = [&](int half, uint32_t scale_own) {
          // everything is read before anything is stored: the compiler keeps reads behind stores that it
          // cannot tell apart from them
          uint2 codes[4][2];
          uint32_t scale_row[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            codes[j][0] = *reinterpret_cast<const uint2*>(raw + half * 2048 + j * 512 + lane * 16 + flip * 8);
            codes[j][1] = *reinterpret_cast<const uint2*>(raw + half * 2048 + j * 512 + lane * 16 + (flip ^ 1) * 8);
            scale_row[j] = __shfl_sync(0xffffffffu, scale_own, half * 16 + 4 * j + sub);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint8_t* to_row = wide + st * kTileBytes + half * 2048 + j * 512;
            const int key = (4 * j + sub) & 7;           // the swizzle
            *reinterpret_cast<uint4*>(to_row + ((c0 ^ key) << 4)) = widen8(codes[j][0], scale_row[j]);
            *reinterpret_cast<uint4*>(to_row + ((c0 ^ 1 ^ key) << 4)) = widen8(codes[j][1], scale_row[j]);
          }
        };
        // A group of copies a half, empty ones too.  The first half's holds the exponents of both and the
        // entries of the group's next position.
        if (i0 < n) {
          ask(i0);
          asm volatile("cp.async.wait_all;" ::: "memory");
          asked(i0);
          fetch_exps();
          fetch_half(0);
          ask(i0 + kGroups);
          asm volatile("cp.async.commit_group;" ::: "memory");
          fetch_half(1);
          asm volatile("cp.async.commit_group;" ::: "memory");
        }
        int i = i0;
        for (; i < n; i += kGroups) {
          ok = wait_to_fill([&](bool filled) {
            return warp_wait(filled ? &ctl.kv_full[st] : &ctl.kv_empty[st], phase, abort_flag);
          });
          if (!ok) break;
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          const uint32_t scale_own = scale_pair(raw[L::kRawExps + lane * 16 + bytes]);
          store_half(0, scale_own);
          const bool more = i + kGroups < n;
          asked(i + kGroups);                            // from here on row, is_v and bytes are the next position's
          if (more) {
            fetch_exps();
            fetch_half(0);
            ask(i + 2 * kGroups);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          store_half(1, scale_own);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.kv_full[st]);
          st += kGroups;
          if (st >= static_cast<uint32_t>(stages)) st -= stages, phase ^= 1u;
          if (more) fetch_half(1);
          asm volatile("cp.async.commit_group;" ::: "memory");
        }
        own = i - n;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");   // nothing in flight when the CTA leaves
  } else if (warp < kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kControlRegs));

    if (warp == kPlanWarp && lane == 0) {
      // ---- the units of this part, in order, and their query tiles
      long long cur = lo, req_pos = ctl.start_pos;
      int b = ctl.start_b, it = 0, toggle = 0;
      uint32_t q_uses[2] = {0u, 0u};
      bool ok = true;
      const uint32_t q_bytes = static_cast<uint32_t>(tile_tokens) * G * 128u;   // of one 64-dim half
      while (ok && cur < hi) {
        const Request r = load_request(a, b, false);
        const long long len = head_cells(r, a.window, span);
        if (cur >= req_pos + len * a.Hkv) {
          req_pos += len * a.Hkv;
          ++b;
          continue;
        }
        int kh = static_cast<int>((cur - req_pos) / len), t = 0;
        long long u0 = req_pos + kh * len;
        Unit u = unit_of(r, a.window, span, 0);
        while (cur >= u0 + cells_of(u)) {
          u0 += cells_of(u);
          u = unit_of(r, a.window, span, ++t);
        }
        while (ok && cur < hi && kh < a.Hkv) {
          const Unit now = u;
          const long long first = u0 + kUnitCells, u1 = u0 + cells_of(now);
          const long long from = max(cur, first), to = min(hi, u1);
          const int tok0 = r.row0 + now.t0, head = kh;
          const bool begins = cur <= u0;
          cur = max(cur, to);
          u0 = u1;
          if (++t * span >= r.n) {
            t = 0;
            ++kh;
          }
          u = unit_of(r, a.window, span, t);
          if (now.nblk > 0 ? from >= to : !begins) continue;   // no block of it in this part
          const int slot = it & (kItems - 1);
          ok = mbar_wait(&ctl.item_empty[slot], (it / kItems) + 1, abort_flag);
          if (!ok) break;
          Item& o = ctl.items[slot];
          o.valid = 1;
          o.dual = now.ntok > tile_tokens;
          o.kh = head;
          o.req = r.req;
          o.tok0 = tok0;
          o.ntok = now.ntok;
          o.pos0 = r.kv - r.n + now.t0;
          o.k0 = now.k0;
          o.khi = now.khi;
          o.blk0 = static_cast<int>(from - first);
          o.nblk = now.nblk == 0 ? 0 : static_cast<int>(to - from);
          o.qbuf = toggle;
          o.parts = 1;
          o.slot = 0;
          if (now.nblk > 0) {                            // the CTAs of its first and last block
            const int cta0 = static_cast<int>(((first + 1) * ctas - 1) / total);
            o.parts = static_cast<int>((u1 * ctas - 1) / total) - cta0 + 1;
            const bool first_part = cta0 == static_cast<int>(blockIdx.x);
            o.slot = 2 * static_cast<int>(blockIdx.x) + (first_part ? 1 : 0);
            if (first_part && o.parts > 1) cuts[blockIdx.x] = Cut{o.parts, head, tok0, now.ntok};
          }
          o.nonfinite = 0u;
          const int dual = o.dual, nblk = o.nblk;
          mbar_arrive(&ctl.item_full[slot]);
          if (nblk > 0) {
            for (int i = 0; i < (dual ? 2 : 1) && ok; ++i) {
              const int buf = dual ? i : toggle;
              ok = mbar_wait(&ctl.q_empty[buf], q_uses[buf] + 1, abort_flag);
              if (!ok) break;
              ++q_uses[buf];
              mbar_expect_tx(&ctl.q_full[buf], 2 * q_bytes);
              const uint32_t dst = smem_u32(smem + kSmemQ + buf * kTileBytes);
              tma_load_3d(dst, &q_map, 0, head * G, tok0 + i * tile_tokens, &ctl.q_full[buf]);
              tma_load_3d(dst + kHalfBytes, &q_map, 64, head * G, tok0 + i * tile_tokens, &ctl.q_full[buf]);
            }
            if (!dual && stages == kStages) toggle ^= 1;
          }
          ++it;
        }
      }
      const int slot = it & (kItems - 1);
      if (ok && mbar_wait(&ctl.item_empty[slot], (it / kItems) + 1, abort_flag)) {
        ctl.items[slot].valid = 0;
        mbar_arrive(&ctl.item_full[slot]);
      }
      // a query tile still on its way when the CTA gives up must land before the CTA leaves
      if (*reinterpret_cast<volatile unsigned*>(abort_flag) != 0u)
        for (int i = 0; i < 2; ++i) {
          const long long t0 = clock64();
          while (q_uses[i] > 0 && !mbar_try(smem_u32(&ctl.q_full[i]), (q_uses[i] - 1) & 1u) &&
                 clock64() - t0 < kWaitLimitClocks) {}
        }
    } else if (warp < kMmaWarp + 2) {
      // ---- the products of stream `warp - kMmaWarp`.  The whole warp walks through the steps and one
      // lane issues: in code that the compiler knows to be uniform the operands' descriptors stay in
      // uniform registers (a lane that branched off by itself took 90 cycles an instruction).  One
      // warp a stream: neither waits for the other's softmax.
      const int s = warp - kMmaWarp;
      const uint32_t t_s = tmem + s * 128, t_o = tmem + 256 + s * 128;
      // What one warp computes between two products is latency on the tensor cores' path: stages and
      // phases are counted along, not divided out of positions, and descriptors are sums.
      uint32_t q_phase[2] = {0u, 0u}, t = 0;             // t: steps of 64 keys so far
      uint32_t st = 0, phase = 0;                        // of the ring position to wait for next
      const uint64_t desc_q = operand_desc(smem_u32(smem + kSmemQ), 16);
      const uint64_t desc_k = operand_desc(smem_u32(ring), 16);
      const uint64_t desc_v = operand_desc(smem_u32(ring), kHalfBytes);
      constexpr uint64_t kDescTile = kTileBytes >> 4, kDescHalf = (kHalf * 128) >> 4;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const int slot = it & (kItems - 1);
        ok = warp_wait(&ctl.item_full[slot], it / kItems, abort_flag);
        if (!ok) break;
        const Item& o = ctl.items[slot];
        if (!uniform(o.valid)) break;
        const int dual = uniform(o.dual), nblk = uniform(o.nblk), qbuf = uniform(o.qbuf);
        const int keys = uniform(o.khi - o.k0 - o.blk0 * kBlk);
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.item_empty[slot]);
        if (nblk == 0) continue;
        const int n = dual ? nblk : (nblk + 1 - s) >> 1;  // blocks of this stream
        const int buf = dual ? s : qbuf;
        // A barrier tells its phases apart by one bit, so no phase may pass a waiter by: both streams'
        // warps wait for every ring position in order, and each gives every position back -- with its
        // last product on it, or at once when the block is the other stream's.  The same for query
        // tiles.
        for (int i = 0; i < 2; ++i)
          if (dual || i == qbuf) {
            ok = ok && warp_wait(&ctl.q_full[i], q_phase[i], abort_flag);
            q_phase[i] ^= 1u;
            if ((i != buf || n == 0) && lane == 0) mbar_arrive(&ctl.q_empty[i]);
          }
        int at = 0, k_next = 0, v_next = 0;              // positions of the unit waited for; single: K, V blocks
        // waits for the stream's next own position; its stage, or -1
        auto next_stage = [&]() {
          while (ok) {
            ok = warp_wait(&ctl.kv_full[st], phase, abort_flag);
            bool mine = true;
            if (!dual) {
              const bool is_v = k_next == nblk || k_next > v_next + 1;
              mine = ((is_v ? v_next++ : k_next++) & 1) == s;
              if (!mine && lane == 0) mbar_arrive(&ctl.kv_empty[st]);
            }
            const int found = static_cast<int>(st);
            ++at;
            if (++st == stages) st = 0, phase ^= 1u;
            if (mine) return found;
          }
          return -1;
        };
        const uint64_t dq = desc_q + buf * kDescTile;
        // The last block may hold one half only.  Scores run two steps ahead of the weights: step t
        // takes score buffer t & 1, and its weights lie where its scores were.
        const int steps = 2 * n - (n > 0 && keys - (dual ? n - 1 : 2 * (n - 1) + s) * kBlk <= kHalf ? 1 : 0);
        int st_k = 0, st_v = 0;
        const uint32_t t0 = t;
        auto pv = [&](int i) {                           // O += P V of step i
          if (!ok || i < 0 || i >= steps) return;
          const int h = i & 1;
          const uint32_t b = t & 1;
          if (h == 0) st_v = next_stage();
          ok = ok && warp_wait(&ctl.p_full[s][b], t >> 1, abort_flag);
          if (!ok) return;
          ++t;
          fence_async_smem();
          tc_fence_after();
          const uint64_t dv = desc_v + uniform(st_v) * kDescTile + h * kDescHalf;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)                  // 16 keys each: two eight-row groups of V
              mma_ts(t_o, t_s + b * kHalf + k * 8, dv + static_cast<uint64_t>(k * 2048 >> 4), i > 0 || k > 0);
            mma_commit(&ctl.o_done[s][b]);
            if (h == 1 || i == steps - 1) mma_commit(&ctl.kv_empty[st_v]);
          }
          __syncwarp();
        };
        auto qk = [&](int i) {                           // S = Q K^T of step i, into the buffer just emptied
          if (!ok || i >= steps) return;
          const int h = i & 1;
          const uint32_t b = (t0 + i) & 1;
          // The weights of two steps ago lie where these scores go, and the product that reads them has
          // another shape and accumulator: issued before, but not promised to run before.
          ok = warp_wait(&ctl.o_done[s][b], (t0 + i + 2) >> 1, abort_flag);
          if (h == 0) st_k = next_stage();
          if (!ok) return;
          fence_async_smem();
          tc_fence_after();
          const uint64_t dk = desc_k + uniform(st_k) * kDescTile + h * kDescHalf;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint64_t off = static_cast<uint64_t>(((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4);
              mma_ss(t_s + b * kHalf, dq + off, dk + off, k > 0);
            }
            mma_commit(&ctl.s_full[s][b]);
            if (h == 1 || i == steps - 1) mma_commit(&ctl.kv_empty[st_k]);
            if (i == steps - 1) mma_commit(&ctl.q_empty[buf]);
          }
          __syncwarp();
        };
        if (kE4m3 && !dual) {
          // Where the ring is short (three positions, four in a call whose units are all of one tile) and
          // the streams alternate, both products of a block's values come before the scores of the
          // stream's next block: values that wait for the next keys before they are given back hold up
          // the keys behind them.  (The decode call above, four positions: 390 us, 401 in the other
          // order; five positions of bf16 gain nothing by it, 397 us either way.)
          for (int i = 0; ok && steps > 0 && i < steps + 2; i += 2) pv(i - 2), pv(i - 1), qk(i), qk(i + 1);
        } else {
          for (int i = 0; ok && steps > 0 && i < steps + 2; ++i) pv(i - 2), qk(i);
        }
        while (ok && at < 2 * nblk) {                    // the other stream's last positions
          ok = warp_wait(&ctl.kv_full[st], phase, abort_flag);
          if (lane == 0) mbar_arrive(&ctl.kv_empty[st]);
          ++at;
          if (++st == stages) st = 0, phase ^= 1u;
        }
      }
    }
  } else {
    // ---- softmax: this thread's row of its stream
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftmaxRegs));
    const int s = (warp - kSoftmaxWarp) >> 2, r = tid & 127;
    const uint32_t t_lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + s * 128 + t_lane, t_o = tmem + 256 + s * 128 + t_lane;
    const float scale = a.sm_scale * 1.4426950408889634f;
    const float slack = 8.f / scale;                     // scores may exceed the kept maximum by this
    const bool whole_sectors = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0u;
    char* const slots = static_cast<char*>(a.workspace) + kCutBytes;
    uint32_t t = 0, j_uses = 0, pos = 0;                 // t: steps of this stream so far
    bool ok = true;
    auto both_streams = [&]() {                          // barrier of the eight softmax warps, bounded
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.join);
      return warp_wait(&ctl.join, j_uses++, abort_flag);
    };
    for (int it = 0; ok; ++it) {
      const int islot = it & (kItems - 1);
      ok = warp_wait(&ctl.item_full[islot], it / kItems, abort_flag);
      if (!ok) break;
      Item& o = ctl.items[islot];
      if (!o.valid) break;
      const int dual = o.dual, nblk = o.nblk, ntok = o.ntok;
      const int token = (dual ? s * tile_tokens : 0) + r / G;
      const bool live = r < tile_tokens * G && token < ntok;
      const bool any_live = __any_sync(0xffffffffu, live);
      const int p = o.pos0 + token;
      // keys of this row; padding rows take all (they are computed and thrown away)
      const int key_lo = live && a.window >= 0 ? static_cast<int>(max(0ll, static_cast<long long>(p) + 1 - a.window)) : 0;
      const int key_hi = live ? p + 1 : INT_MAX;
      const int first = o.k0 + o.blk0 * kBlk;
      // keys that every row of the warp attends: [warp_lo, warp_hi); steps inside need no mask
      const int warp_lo = __reduce_max_sync(0xffffffffu, key_lo), warp_hi = __reduce_min_sync(0xffffffffu, key_hi);
      // and that every row of the unit does; blocks inside need no look at their values
      const int unit_lo = a.window >= 0 ? o.pos0 + ntok - a.window : 0, unit_hi = o.pos0 + 1, khi = o.khi;
      float m = -INFINITY, l = 0.f;
      const int step = dual ? 1 : 2, blk_first = dual ? 0 : s;
      for (int blk = blk_first; blk < nblk && ok; blk += step) {
       const int kb = first + blk * kBlk, nh = khi - kb > kHalf ? 2 : 1;
       for (int h = 0; h < nh; ++h) {
        const uint32_t b = t & 1, t_sb = t_s + b * kHalf;
        ok = mbar_wait(&ctl.s_full[s][b], t >> 1, abort_flag);   // voted on below, on each way
        tc_fence_after();
        if (h == 0 && (min(kb + kBlk, khi) > unit_hi || kb < unit_lo)) {
          // A weight of zero does not silence an infinite or NaN value in the product.  Such values
          // of a block that some rows attend only in part are taken out here and put back, for the
          // rows that do attend them, when the unit ends.
          const uint32_t vp = pos + ring_v(dual, blk, nblk), st = vp % stages;
          ok = __all_sync(0xffffffffu, ok) && warp_wait(&ctl.kv_full[st], vp / stages, abort_flag);
          if (!ok) break;
          uint32_t* v = reinterpret_cast<uint32_t*>(ring + st * kTileBytes);
          unsigned found = 0;
#pragma unroll 4
          for (int i = 0; i < kTileBytes / 16 / 128; ++i) {
            const uint4 w4 = *reinterpret_cast<const uint4*>(v + (i * 128 + r) * 4);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              found |= ((w[j] & 0x7f80u) == 0x7f80u || (w[j] & 0x7f800000u) == 0x7f800000u) ? 1u : 0u;
          }
          if (found) {
            *reinterpret_cast<volatile unsigned*>(&o.nonfinite) = 1u;   // before any value is taken out
            __threadfence_block();
#pragma unroll 1
            for (int i = 0; i < kTileBytes / 16 / 128; ++i) {
              const uint32_t at = smem_u32(v + (i * 128 + r) * 4);
              uint32_t w[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                           : "r"(at)
                           : "memory");
              // one store a word, and the last word on it: see finite_halves()
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(finite_halves(w[0])),
                           "r"(finite_halves(w[1])), "r"(finite_halves(w[2])), "r"(finite_halves(w[3]))
                           : "memory");
            }
          }
          fence_async_smem();
          __syncwarp();                                  // the tensor-memory instructions want whole warps
        }
        if (!any_live) {                                 // rows that nobody reads: any weights will do
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_arrive(&ctl.p_full[s][b]);
          __syncwarp();
          ++t;
          continue;
        }
        uint32_t u[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld32(t_sb + c * 32, u[c]);
        tmem_ld_wait();
        loaded(u[0]);
        loaded(u[1]);
        const int ks = kb + h * kHalf;
        const int c_lo = key_lo - ks, c_hi = key_hi > ks + kHalf ? kHalf : key_hi - ks;   // columns in [c_lo, c_hi)
        if (ks < warp_lo || ks + kHalf > warp_hi) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i < c_lo || c * 32 + i >= c_hi) u[c][i] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t* x = &u[c >> 1][(c & 1) * 16];
          mx[c] = max3(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
#pragma unroll
          for (int i = 3; i < 15; i += 2) mx[c] = max3(mx[c], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
        }
        mx[0] = max3(mx[0], __uint_as_float(u[0][15]), __uint_as_float(u[0][31]));
        mx[1] = max3(mx[1], __uint_as_float(u[1][15]), __uint_as_float(u[1][31]));
        const float bm = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
        const bool grow = bm > m + slack || (m == -INFINITY && bm > m);
        if (__any_sync(0xffffffffu, grow || !ok)) {
          if (!__all_sync(0xffffffffu, ok)) {            // the wait for the scores gave up
            ok = false;
            break;
          }
          const float f = !grow ? 1.f : m == -INFINITY ? 0.f : ex2((m - bm) * scale);
          if (grow) m = bm;
          l *= f;
          if (blk != blk_first || h > 0) {
            // the product of the step before has to be in
            ok = warp_wait(&ctl.o_done[s][b ^ 1], (t - 1) >> 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t w[32];
              tmem_ld32(t_o + c * 32, w);
              tmem_ld_wait();
              loaded(w);
#pragma unroll
              for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * f);
              tmem_st32(t_o + c * 32, w);
            }
          }
        }
        // A logit of NaN or +inf makes the row NaN from here on (softmax of it is NaN).
        if (!(bm < INFINITY)) m = __uint_as_float(0x7fc00000u);
        const float ms = m == -INFINITY ? 0.f : m * scale;
        const uint64_t scale2 = pair(scale, scale), ms2 = pair(-ms, -ms);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float e0, e1;
            unpair(fma2(pair(__uint_as_float(u[c][2 * i]), __uint_as_float(u[c][2 * i + 1])), scale2, ms2), e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            u[c][2 * i] = __float_as_uint(e0);
            u[c][2 * i + 1] = __float_as_uint(e1);
            w[i] = pack_bf16(e0, e1);
          }
          tmem_st16(t_sb + c * 16, w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full[s][b]);
        uint64_t sum[2] = {0ull, 0ull};                  // while the product runs
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sum[c] = add2(sum[c], pair(__uint_as_float(u[c][2 * i]), __uint_as_float(u[c][2 * i + 1])));
        float l0, l1;
        unpair(add2(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
        ++t;
       }
      }
      if (!ok) break;
      pos += 2 * nblk;
      // ---- the unit's (part's) result.  Dual: a thread's own row.  Single: both streams hold a share
      // of every row; stream 0 finishes dims 0-63 and stream 1 dims 64-127.
      if (blk_first < nblk) {
        ok = warp_wait(&ctl.o_done[s][(t - 1) & 1], (t - 1) >> 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      float fa = 1.f, fb = 0.f;                          // what the accumulators are multiplied by
      if (!dual) {
        ctl.ml[s][r] = make_float2(m, l);
        tc_fence_before();
        ok = both_streams();                             // the other stream's results are there too
        if (!ok) break;
        const float2 x = ctl.ml[0][r], y = ctl.ml[1][r];
        m = fmaxf(x.x, y.x);
        fa = x.x == -INFINITY ? 0.f : ex2((x.x - m) * scale);
        fb = y.x == -INFINITY ? 0.f : ex2((y.x - m) * scale);
        // a NaN sum has to survive a maximum of -inf (every logit NaN)
        l = (x.y == 0.f ? 0.f : x.x == -INFINITY ? x.y : x.y * fa) +
            (y.y == 0.f ? 0.f : y.x == -INFINITY ? y.y : y.y * fb);
      }
      tc_fence_after();
      __threadfence_block();
      const bool refill = *reinterpret_cast<volatile unsigned*>(&o.nonfinite) != 0u;
      const bool cut = o.parts > 1;
      const int64_t orow = static_cast<int64_t>(o.tok0 + token) * a.Hq + o.kh * G + r % G;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      float* const part = reinterpret_cast<float*>(slots + static_cast<int64_t>(o.slot) * kSlotBytes);
      const int prow = dual ? s * kRows + r : r;
      const uint32_t t_a = dual ? t_o : tmem + 256 + t_lane;
      if (any_live) {
#pragma unroll 1
        for (int c = dual ? 0 : 2 * s; c < (dual ? 4 : 2 * s + 2); ++c) {
          float v[32];
          __syncwarp();
          if (nblk > 0) {
            uint32_t w[32];
            tmem_ld32(t_a + c * 32, w);
            tmem_ld_wait();
            loaded(w);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(w[i]) * fa;
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
          }
          if (!dual && nblk > 1) {
            uint32_t w[32];
            tmem_ld32(t_a + 128 + c * 32, w);
            tmem_ld_wait();
            loaded(w);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = fmaf(__uint_as_float(w[i]), fb, v[i]);
          }
          if (refill && live) {
            for (int blk = 0; blk < nblk; ++blk) {
              const int kb = first + blk * kBlk;
              if (min(kb + kBlk, khi) <= unit_hi && kb >= unit_lo) continue;
              for (int key = max(kb, key_lo); key < min(kb + kBlk, key_hi); ++key) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float2 x = value_pair<kE4m3>(a, o, key, c * 32 + 2 * i);
                  if (!isfinite(x.x)) v[2 * i] += x.x;
                  if (!isfinite(x.y)) v[2 * i + 1] += x.y;
                }
              }
            }
          }
          if (live && !cut) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(a.out) + orow * 256 + c * 64);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t w[8];
#pragma unroll
              for (int j = 0; j < 8; ++j)
                w[j] = l == 0.f ? 0u : pack_bf16(v[i * 16 + 2 * j] * inv, v[i * 16 + 2 * j + 1] * inv);
              store32(dst + 2 * i, w, whole_sectors);
            }
          } else if (live) {
            float4* dst = reinterpret_cast<float4*>(part) + c * 8 * kSlotRows + prow;   // four dims of all rows
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[i * kSlotRows] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
      }
      if (live && (dual || s == 0)) {
        if (cut)
          reinterpret_cast<float2*>(part + kSlotFloats)[prow] = make_float2(m, l);
        else if (a.lse)
          a.lse[orow] = l == 0.f ? -INFINITY : (m * scale + log2f(l)) * 0.6931471805599453f;
      }
      __syncwarp();
      if (!dual) {
        tc_fence_before();
        ok = both_streams();                             // the accumulators and ctl.ml are free again
        if (!ok) break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.item_empty[islot]);
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && ctl.abort != 0u) atomicOr(&g_chunk_status, ctl.abort);
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---------------------------------------------------------------------- units that were cut
// Block (c, y) joins rows [16 y, 16 y + 16) of the unit that begins in part c.  A thread owns eight
// dims of a row; where the rows leave threads free, the parts are shared among them too.  The sums
// run in an order that the parts and rows alone decide.
__global__ void __launch_bounds__(256)
chunk_join_kernel(const MacB200ChunkArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Cut cut = static_cast<const Cut*>(a.workspace)[blockIdx.x];
  const int G = a.Hq / a.Hkv, tile_tokens = kRows / G;
  const int row_first = blockIdx.y * kJoinRows, rows = min(cut.ntok * G - row_first, kJoinRows);
  if (cut.parts == 0 || rows <= 0) return;
  __shared__ float4 acc_s[2][256];
  __shared__ float l_s[256];
  const int tid = threadIdx.x;
  const int width = rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows;   // rows rounded up to a power of two
  const int groups = 16 / width;                         // that share the parts
  const int rr = tid % width, k = tid / width % 16, group = tid / (width * 16);
  const char* const slots = static_cast<const char*>(a.workspace) + kCutBytes;
  const float scale = a.sm_scale * 1.4426950408889634f;
  const int row = row_first + min(rr, rows - 1);
  const int token = row / G, g = row - token * G;
  const bool second = cut.ntok > tile_tokens && token >= tile_tokens;
  const int at = second ? row - tile_tokens * G + kRows : row;
  auto slot_of = [&](int i) {
    return slots + static_cast<int64_t>(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * kSlotBytes;
  };
  float mx = -INFINITY;
#pragma unroll 8
  for (int i = group; i < cut.parts; i += groups)
    mx = fmaxf(mx, reinterpret_cast<const float2*>(slot_of(i) + kSlotFloats * 4)[at].x);
  if (groups > 1) {
    l_s[tid] = mx;
    __syncthreads();
    for (int i = 0; i < groups; ++i) mx = fmaxf(mx, l_s[i * width * 16 + k * width + rr]);
    __syncthreads();
  }
  const float ms = mx == -INFINITY ? 0.f : mx * scale;
  float l = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
  for (int i = group; i < cut.parts; i += groups) {
    const char* sl = slot_of(i);
    const float2 ml = reinterpret_cast<const float2*>(sl + kSlotFloats * 4)[at];
    const float4* x = reinterpret_cast<const float4*>(sl) + at;
    const float4 x0 = x[k * kSlotRows], x1 = x[(k + 16) * kSlotRows];
    if (ml.y != 0.f) {                                   // something attended in this part
      const float f = ml.x == -INFINITY ? 1.f : ex2(ml.x * scale - ms);   // NaN sums stay
      l += ml.y * f;
      acc[0].x += x0.x * f, acc[0].y += x0.y * f, acc[0].z += x0.z * f, acc[0].w += x0.w * f;
      acc[1].x += x1.x * f, acc[1].y += x1.y * f, acc[1].z += x1.z * f, acc[1].w += x1.w * f;
    }
  }
  if (groups > 1) {
    acc_s[0][tid] = acc[0];
    acc_s[1][tid] = acc[1];
    l_s[tid] = l;
    __syncthreads();
    if (group != 0) return;
    for (int i = 1; i < groups; ++i) {
      const int t = i * width * 16 + tid;
      l += l_s[t];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 x = acc_s[h][t];
        acc[h].x += x.x, acc[h].y += x.y, acc[h].z += x.z, acc[h].w += x.w;
      }
    }
  }
  if (rr >= rows) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t to = static_cast<int64_t>(cut.tok0 + token) * a.Hq + cut.kh * G + g;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint2 w = make_uint2(0u, 0u);
    if (l != 0.f)
      w = make_uint2(pack_bf16(acc[h].x * inv, acc[h].y * inv), pack_bf16(acc[h].z * inv, acc[h].w * inv));
    *reinterpret_cast<uint2*>(static_cast<char*>(a.out) + to * 256 + (k + 16 * h) * 8) = w;
  }
  if (a.lse && k == 0) a.lse[to] = l == 0.f ? -INFINITY : (ms + log2f(l)) * 0.6931471805599453f;
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int64_t workspace_bytes(int sms) { return kCutBytes + 2 * static_cast<int64_t>(sms) * kSlotBytes; }

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeTiledFn>(ptr);
  }();
  return fn;
}

// Sets the kernel up on the current device, once: its shared memory, and the check that it was
// built with the registers that its warps trade among themselves (a build with fewer would wait
// for them for ever).
template <bool kE4m3>
int prepare_kernel(int device) {
  static std::atomic<int> ready[64];
  if (device >= 0 && device < 64 && ready[device].load(std::memory_order_acquire)) return MAC_B200_OK;
  cudaFuncAttributes attr{};
  MAC_CUDA(cudaFuncGetAttributes(&attr, chunk_attention_kernel<kE4m3>));
  if (attr.numRegs < Layout<kE4m3>::kLaunchRegs)
    return fail(MAC_B200_EUNSUPPORTED, "the chunk attention kernel was built with %d registers a thread",
                attr.numRegs);
  MAC_CUDA(cudaFuncSetAttribute(chunk_attention_kernel<kE4m3>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Layout<kE4m3>::kBytes));
  if (device >= 0 && device < 64) ready[device].store(1, std::memory_order_release);
  return MAC_B200_OK;
}

int chunk_attention(const MacB200ChunkArgs* args, bool e4m3, void* stream_v) {
  MAC_REQUIRE(args != nullptr, "chunk args must not be null");
  MacB200ChunkArgs a = *args;
  if (a.window >= (1 << 30)) a.window = -1;              // longer than any cache
  MAC_REQUIRE(a.D == 128, "chunk attention needs D=128");
  MAC_REQUIRE(a.Hq > 0 && a.Hkv > 0 && a.Hq % a.Hkv == 0 && a.Hq / a.Hkv <= 16,
              "Hq must be Hkv times 1..16");
  MAC_REQUIRE(a.Hkv <= 1024, "Hkv must not exceed 1024");
  MAC_REQUIRE(a.B >= 0 && a.q_rows >= 0, "negative batch");
  MAC_REQUIRE(a.B < (1 << 30) && a.q_rows < (1 << 30), "batch too large");
  MAC_REQUIRE(std::isfinite(a.sm_scale) && a.sm_scale > 0.f, "sm_scale must be positive");
  if (a.B == 0 || a.q_rows == 0) return MAC_B200_OK;
  MAC_REQUIRE(a.q && a.k && a.v && a.req_to_token && a.req_ids && a.offsets && a.kv_lens && a.out && a.workspace,
              "chunk tensors must not be null");
  MAC_REQUIRE(!e4m3 || (a.k_exp && a.v_exp), "the 8-bit pool needs its exponents");
  MAC_REQUIRE(a.kv_tokens > 0 && a.kv_tokens < (int64_t(1) << 31), "the pool must hold 1..2^31-1 rows");
  MAC_REQUIRE(a.req_to_token_rows > 0 && a.req_to_token_stride > 0, "req_to_token must not be empty");
  MAC_REQUIRE(a.req_to_token_stride < (1 << 30), "req_to_token rows are too long");
  MAC_REQUIRE(a.q_stride0 < (int64_t(1) << 38), "q row stride too large");
  MAC_REQUIRE(a.q_stride0 >= static_cast<int64_t>(a.Hq) * 128 && a.q_stride0 % 8 == 0,
              "q row stride must be a multiple of 8 and at least Hq*128");
  MAC_REQUIRE(on16(a.q) && on16(a.k) && on16(a.v) && on16(a.out) && on16(a.workspace),
              "chunk tensors must be 16-byte aligned");
  const int64_t out_bytes = a.q_rows * static_cast<int64_t>(a.Hq) * 256;
  MAC_REQUIRE(!byte_ranges_meet(a.q, (a.q_rows - 1) * a.q_stride0 * 2 + a.Hq * int64_t{256}, a.out, out_bytes),
              "q and out must not share memory");
  int device = 0;
  MAC_CUDA(cudaGetDevice(&device));
  const int sms = device_sm_count(device);
  MAC_REQUIRE(a.workspace_bytes >= workspace_bytes(sms), "workspace holds %lld bytes, %lld are needed",
              static_cast<long long>(a.workspace_bytes), static_cast<long long>(workspace_bytes(sms)));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  MAC_REQUIRE(sms <= kMaxCtas, "too many multiprocessors");
  if (const int rc = e4m3 ? prepare_kernel<true>(device) : prepare_kernel<false>(device)) return rc;
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return fail(MAC_B200_EUNSUPPORTED, "cuTensorMapEncodeTiled is not available");
  alignas(64) CUtensorMap q_map;                         // box: 64 dims x the G heads of a KV head x 128/G tokens
  const cuuint32_t ones[3] = {1u, 1u, 1u};
  const int G = a.Hq / a.Hkv;
  const cuuint64_t q_dims[3] = {128u, static_cast<cuuint64_t>(a.Hq), static_cast<cuuint64_t>(a.q_rows)};
  const cuuint64_t q_strides[2] = {256u, static_cast<cuuint64_t>(a.q_stride0) * 2};
  const cuuint32_t q_box[3] = {64u, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(kRows / G)};
  const CUresult rc = enc(&q_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), q_dims, q_strides,
                          q_box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(MAC_B200_ECUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(rc));
  if (e4m3)
    chunk_attention_kernel<true><<<sms, Layout<true>::kThreads, Layout<true>::kBytes, stream>>>(a, q_map);
  else
    chunk_attention_kernel<false><<<sms, Layout<false>::kThreads, Layout<false>::kBytes, stream>>>(a, q_map);
  MAC_CUDA(cudaGetLastError());
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  cudaLaunchConfig_t config{};
  const int most_rows = std::min(a.q_rows, 2 * (kRows / G)) * G;   // of a unit
  config.gridDim = dim3(static_cast<unsigned>(sms), static_cast<unsigned>((most_rows + kJoinRows - 1) / kJoinRows));
  config.blockDim = dim3(256);
  config.stream = stream;
  cudaLaunchAttribute early{};                           // set up while the first kernel runs
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  MAC_CUDA(cudaLaunchKernelEx(&config, chunk_join_kernel, a));
  MAC_CUDA(cudaGetLastError());
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  return MAC_B200_OK;
}

}  // namespace

int chunk_status_word(unsigned** word) {
  MAC_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(word), g_chunk_status));
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
