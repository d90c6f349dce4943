// Fifth-generation tensor core plumbing for sm_100a: TMEM allocation and reads, the block-scaled matrix product
// (tcgen05.mma kind::mxf8f6f4), the copies of its scales into TMEM, and waits that end.
//
// Every wait is bounded in time and also ends when another role of the CTA has given up: the first wait
// that runs out raises the CTA's `abort` word in shared memory, every later wait returns false at once, and the roles
// leave their loops together.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tma.cuh"

namespace mxq {
namespace tc {

// how many cycles a wait may take, about two seconds: a correct one takes microseconds
constexpr long long kWaitCycles = 4000000000ll;

// PAIR: what the barrier's arrivals in the other CTA of the pair released is seen by this thread too
template <bool PAIR>
__device__ __forceinline__ bool try_wait(uint64_t* bar, unsigned parity) {
  if (!PAIR) return mbar_try_wait_rounds(bar, parity, 1);
  unsigned done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done;
}

// What bounds a CTA's waits: its word in shared memory, the library's status word, the limit.
struct Guard {
  volatile int* abort;
  unsigned* status;
  long long cycles;
};
// false: gave up (this wait ran out, or another role's did)
template <bool PAIR>
__device__ __forceinline__ bool wait(uint64_t* bar, unsigned parity, const Guard& g) {
  if (try_wait<PAIR>(bar, parity) || try_wait<PAIR>(bar, parity)) return true;
  const long long begin = clock64();
  do {
    if (try_wait<PAIR>(bar, parity) || try_wait<PAIR>(bar, parity)) return true;
    if (*g.abort) return false;
  } while (clock64() - begin < g.cycles);
  *g.abort = 1;
  note_wait_timeout(g.status);
  return false;
}
// the same for what a role that gave up has in flight towards shared memory or TMEM, without the abort word
__device__ __forceinline__ void settle(uint64_t* bar, unsigned parity, const Guard& g) {
  const long long begin = clock64();
  while (!try_wait<false>(bar, parity) && clock64() - begin < g.cycles / 16) {
  }
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_addr(bar)) : "memory");
}
// wait() by a whole warp: the answer is the same in every lane, and the compiler knows it
template <bool PAIR>
__device__ __forceinline__ bool wait_warp(uint64_t* bar, unsigned parity, const Guard& g) {
  return __all_sync(0xffffffffu, wait<PAIR>(bar, parity, g));
}
// one lane of a converged warp. The operands of what it issues have to be warp-uniform for the compiler (no lane index
// in them, no branch on one around them): tcgen05 and TMA instructions take uniform registers, and from a branch on
// the lane each of their operands is moved there one by one, about 65 cycles per instruction.
__device__ __forceinline__ bool elect() {
  unsigned yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
  return yes;
}

// the same barrier in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
// an arrival there that releases what this thread has written or been told of to the cluster
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// The same word without a release: for what tcgen05.fence::before_thread_sync orders (loads from TMEM that are done), nothing
// in memory.
__device__ __forceinline__ void mbar_word_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

// one whole warp (PAIR: one of each CTA of the pair); the address lands in shared memory
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t cols) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(where)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(where)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  if (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(addr), "r"(cols));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(addr), "r"(cols));
}

// Programmatic dependent launch: this kernel may have been launched while the one before it on the stream was still
// at work; what that one (or any before it) wrote may be read after this. TMEM is allocated after it too: held while
// waiting, it could be what a block of the kernel before still needs to go on.
__device__ __forceinline__ void wait_for_prior_grid() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
// The next grid on the stream, if it waits as above, may be launched from here on: every block of this one has its TMEM, and
// the launch and the set-up of the next (0.5 us of a small product's 7) pass beside this one's work.
__device__ __forceinline__ void start_next_grid() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}

// K-major operand tile, rows of 128 bytes in the 128-byte swizzle: groups of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// 32 rows of 16 bytes, no swizzle: groups of 8 rows 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | (8ull << 32) | (1ull << 46);
}

// instruction descriptor of kind::mxf8f6f4 (K-major A and B, E8M0 scales): operand formats as mma_format() gives
// them, tile m x n, the byte of each scale word that this K step of 32 reads
enum { kE4M3 = 0, kE5M2 = 1, kE2M1 = 5 };
__host__ __device__ constexpr uint32_t mma_desc(int fa, int fb, int m, int n) {
  return ((uint32_t)fa << 7) | ((uint32_t)fb << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t mma_desc_step(uint32_t d, uint32_t byte) { return d | (byte << 4) | (byte << 29); }

// 128 rows' scale words (4 E8M0 bytes each, shared memory (row % 32) * 16 + (row / 32) * 4) into 4 TMEM columns. PAIR:
// in both CTAs, each from its own shared memory.
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(desc) : "memory");
}

// PAIR: 256 rows of A, 128 in each CTA, which also holds half of B's rows; D's rows are in the CTA of their A rows
template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                    bool accumulate) {
  if (PAIR)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"((unsigned)accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"((unsigned)accumulate)
        : "memory");
}
// the barrier (PAIR: of both CTAs) arrives when every tcgen05 operation that this thread has issued is done
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
                     smem_addr(bar)),
                 "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_addr(bar)) : "memory");
}

// 32 columns of this warp's 32 lanes (the lane quarter warp % 4), one row per thread; the wait stands in the same
// statement, so that nothing that uses the values can be moved above it
__device__ __forceinline__ void load32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void load16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      " tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
// loads whose barrier (a shared::cluster address) may be in the other CTA of the pair
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::
          "r"(smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// a box from shared memory to a tensor, under way when it returns; the thread's boxes are read; they are written
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n cp.async.bulk.commit_group;\n" ::"l"(map),
               "r"(x), "r"(y), "r"(smem_addr(src))
               : "memory");
}
__device__ __forceinline__ void store_read() { asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory"); }
__device__ __forceinline__ void store_done() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

// four rows of a tensor, 128 bytes each, one after the other in shared memory
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* map, int x, int4 rows, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
      "%6}], [%7];\n" ::"r"(smem_addr(dst)),
      "l"(map), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(smem_addr(bar))
      : "memory");
}
}  // namespace tc
}  // namespace mxq
