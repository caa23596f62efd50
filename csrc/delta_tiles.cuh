// Matrix tiles of the gated delta rule on the 5th-generation tensor cores, and the pipeline pieces its kernels share.
//
// A tile has rows of 128 bytes (64 16-bit elements) in the 128-byte swizzle: the eight 16-byte pieces of row r lie at places
// piece ^ (r % 8). Wider matrices are panels of 64 columns one behind the other. Tiles lie in global memory as they do in
// shared memory, so that one bulk copy moves each. The same tile is an operand either way: K-major where its rows run
// along the product's rows, MN-major where they run along the summed axis.
//
// A value is held as two bf16 halves in two tiles, hi and lo, which keep 16 bits of its significand; q, k and dO are exact, in
// one bf16 tile or, from fp16, in two.
#pragma once

#include "delta_common.cuh"
#include "tc_common.cuh"

namespace bw {
namespace {

// Parts of an input element: bf16 is its own, fp16 has two.
template <typename I>
constexpr int kParts = 1;
template <>
constexpr int kParts<__half> = 2;

constexpr int kTok = kChunk * 128;  // bytes of a tile of 64 rows

__host__ __device__ constexpr int align1k(int x) { return (x + 1023) / 1024 * 1024; }

// Byte offset of 16-byte piece `piece` (of a panel) of row r.
__device__ __forceinline__ int piece_at(int r, int piece) { return r * 128 + ((piece ^ (r & 7)) << 4); }
// Byte offset of element (r, c) of a tile whose panels are `panel` bytes apart.
__device__ __forceinline__ int element_at(int r, int c, int panel) {
  return (c >> 6) * panel + piece_at(r, (c >> 3) & 7) + (c & 7) * 2;
}

// Two neighbouring values as words of their high and low halves.
__device__ __forceinline__ void halves(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h);
  const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Eight values of a row as one piece of each half's tile.
__device__ __forceinline__ void put8(unsigned char* hi, unsigned char* lo, const float (&x)[8]) {
  uint4 h, l;
  halves(x[0], x[1], h.x, l.x);
  halves(x[2], x[3], h.y, l.y);
  halves(x[4], x[5], h.z, l.z);
  halves(x[6], x[7], h.w, l.w);
  *reinterpret_cast<uint4*>(hi) = h;
  *reinterpret_cast<uint4*>(lo) = l;
}

__device__ __forceinline__ float2 pair_sum(uint32_t hi, uint32_t lo) {
  return make_float2(__uint_as_float(hi << 16) + __uint_as_float(lo << 16),
                     __uint_as_float(hi & 0xffff0000u) + __uint_as_float(lo & 0xffff0000u));
}

template <typename I>
__device__ __forceinline__ const I* head_at(const HeadRows& x, int b, long long t, int h) {
  return reinterpret_cast<const I*>(x.p) + b * x.sb + t * x.st + h * x.sh;
}

// N tokens' values of one column of head rows; zeros behind the last of `rows` tokens. Whole chunks without a condition: with
// one for each load, they wait for one another.
template <typename I, int N>
__device__ __forceinline__ void column_of(const I* p, long long st, int rows, I (&x)[N]) {
  if (rows >= N) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = *p;
      p += st;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = i < rows ? *p : ElemOf<I>::down(0.f);
    p += st;
  }
}

// exp(G_i - G_j) of sums held in two parts: the small part counts where the large ones nearly cancel.
__device__ __forceinline__ float decay_between(float2 i, float2 j) { return __expf((i.x - j.x) + (i.y - j.y)); }

// ---------------------------------------------------------------- products
// Descriptor of a tile in the 128-byte swizzle: groups of eight rows are 1024 bytes apart; `panel` counts for MN-major
// operands of more than 64 rows or columns, whose next 64 lie there.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, int panel) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((panel >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

struct Operand {
  uint32_t addr;  // in shared memory
  int panel;      // bytes between panels
};

constexpr uint32_t kMnA = 1u << 15, kMnB = 1u << 16;

// D (128 x N, from TMEM column d) (+)= A B over 16 kSteps: MN-major operands step 16 rows, K-major ones 16 columns.
template <int kSteps, int N, bool kAmn, bool kBmn>
__device__ __forceinline__ void multiply(uint32_t d, Operand A, Operand B, bool accumulate) {
  constexpr uint32_t idesc = idesc_bf16_f32(128, N) | (kAmn ? kMnA : 0u) | (kBmn ? kMnB : 0u);
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const uint32_t a = A.addr + (kAmn ? k * 2048 : (k >> 2) * A.panel + (k & 3) * 32);
    const uint32_t b = B.addr + (kBmn ? k * 2048 : (k >> 2) * B.panel + (k & 3) * 32);
    tc_mma_f16(d, tile_desc(a, kAmn ? A.panel : 16), tile_desc(b, kBmn ? B.panel : 16), idesc, accumulate || k > 0);
  }
}

// The products of all parts but that of the two low ones; the halves of each lie `lo` bytes apart.
template <int kSteps, int N, bool kAmn, bool kBmn, int kA, int kB>
__device__ __forceinline__ void multiply_parts(uint32_t d, Operand A, int lo_a, Operand B, int lo_b, bool accumulate) {
  multiply<kSteps, N, kAmn, kBmn>(d, A, B, accumulate);
  if (kA == 2) multiply<kSteps, N, kAmn, kBmn>(d, Operand{A.addr + lo_a, A.panel}, B, true);
  if (kB == 2) multiply<kSteps, N, kAmn, kBmn>(d, A, Operand{B.addr + lo_b, B.panel}, true);
}

// The same with B's halves side by side as one operand of twice the columns (they lie `B.panel` apart, or one behind the other):
// D has A's products with either half in N / 2 columns each. An operand A is then read half as often, which is what
// a product of 64 columns waits for.
template <int kSteps, int N, bool kAmn, bool kBmn, int kA>
__device__ __forceinline__ void multiply_wide(uint32_t d, Operand A, int lo_a, Operand B, bool accumulate) {
  multiply<kSteps, N, kAmn, kBmn>(d, A, B, accumulate);
  if (kA == 2) multiply<kSteps, N / 2, kAmn, kBmn>(d, Operand{A.addr + lo_a, A.panel}, B, true);
}

// ---------------------------------------------------------------- copies
__device__ __forceinline__ void bulk_prefetch(const void* from, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)),
               "l"(from), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* to, const void* from, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_u32(from)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_read_done() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_read_one_left() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void bulk_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ---------------------------------------------------------------- tensor memory
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr));
}

// 16 columns of the lane's row.
__device__ __forceinline__ void tmem_row(uint32_t taddr, float (&f)[16]) {
  uint32_t r[16];
  tmem_ld_32x32b_x16(taddr, r);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(r[i]);
}
// Of two matrices at once.
__device__ __forceinline__ void tmem_rows(uint32_t at, float (&f)[16], uint32_t bt, float (&g)[16]) {
  uint32_t r[16], s[16];
  tmem_ld_32x32b_x16(at, r);
  tmem_ld_32x32b_x16(bt, s);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    f[i] = __uint_as_float(r[i]);
    g[i] = __uint_as_float(s[i]);
  }
}

// The sum of two matrices' columns.
__device__ __forceinline__ void tmem_sum(uint32_t at, uint32_t bt, float (&f)[16]) {
  float g[16];
  tmem_rows(at, f, bt, g);
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] += g[i];
}

// Where a worker sits: warp w of sixteen holds tensor memory's lanes 32 (w % 4) .. + 31, one each, and a quarter of the columns.
struct Seat {
  int row, part;
  uint32_t lanes;  // of a tensor memory address
  __device__ Seat() {
    const int warp = threadIdx.x >> 5;
    row = (warp & 3) * 32 + (threadIdx.x & 31);
    part = warp >> 2;
    lanes = (uint32_t)(warp & 3) << 21;
  }
};

// Threads of the sixteen warps that convert (eight leave half of the issue slots empty: a training pass took 8 % longer with them);
// another warp's first lane copies and multiplies.
constexpr int kWorkers = 512, kControl = kWorkers / 32;

// A barrier that completes once in every round of a loop, and its waits. After a wait that gave up the kernel leaves: every
// later wait of the thread returns at once.
struct Waiter {
  int* err;
  bool dead = false;
  __device__ __forceinline__ bool operator()(uint64_t* bar, int round) {
    if (!dead && !mbar_wait(bar, round & 1, err, kErrWaitDone)) dead = true;
    return !dead;
  }
};

// What a worker wrote to shared memory and read or wrote of tensor memory is done before `bar` tells the tensor core so.
__device__ __forceinline__ void hand_over(uint64_t* bar) {
  fence_proxy_async_smem();
  tc_fence_before();
  mbar_arrive(bar);
}

}  // namespace
}  // namespace bw
