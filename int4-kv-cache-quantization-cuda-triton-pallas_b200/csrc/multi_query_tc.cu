// Several 16-bit queries of a sequence over its paged INT4 cache on the 5th
// generation tensor cores: drafted trees and sliding windows in float16 and
// bfloat16 (the float32 form is multi_query_f32.cu).
//
// Math: the logits are taken transposed, S^T[token, row] = K^ Q^T, and so are
// the outputs, O^T[channel, row] += V^T P^T. Tokens and channels fill the 128
// lanes of an MMA whatever the number of rows is, and its cost grows with the
// rows (N = 16, 32, 64 or 128): a handful of drafted rows costs a handful of
// columns, where rows in the lanes would pay for 128. An MMA with few columns is
// bound by the shared memory its 128-lane operand is read from (42 cycles at N =
// 16, 67 at 128, measured), so the dequantized keys never go there: they are
// written to tensor memory, the other place that operand may come from. A thread
// of the softmax holds four tokens and up to 16 rows of a tile (the layout of mma
// fragments), so a row's reference and sum of weights stay in its registers until
// the stream ends. The running maximum is
// kept lazily: weights are 2^(x - ref) against a reference that is raised to the
// true maximum only when some logit exceeds it by more than 14 (in log2), so the
// outputs are rescaled a few times per stream instead of every tile; sums and
// outputs are float32 in registers and tensor memory.
//
// Numerics: keys are dequantized as code * s - zp * s in float32 and rounded once to
// float16 (relative step 2^-11; bfloat16 would lose 3 bits of the logits); queries
// and drafted keys are exact there. What lies outside float16's range is scaled by
// a power of two first, cached keys by group, drafted ones and queries each by its
// own, where the largest magnitude is not in [2^-8, 2^15): inside it what is lost to
// float16's smallest step is 2^-17 of that magnitude at most. The scales return in
// the float32 logits. Weights are rounded to the value pool's type, which the
// tensor cores multiply with the stored values as they are.
//
// A tile is 128 cached tokens (8 pages) or the drafts. Roles of the warps:
//   softmax (a warpgroup for up to 32 rows): S^T from tensor memory, mask, weights
//       to shared memory, the rare rescale of O^T, and the stream's epilogue
//   conversion (two warpgroups, a tile each in turn): packed codes, copied a tile
//       ahead, to float16 keys, a thread a token; a stream's queries; drafted
//       keys. A tile's way through a group is a chain of waits, loads and
//       arithmetic; two chains side by side keep the arithmetic busy.
//   MMA issue (2): S^T, and O^T. Each product waits for its own operands: one warp
//       that issued both in turn was what a tile of 64 or 128 rows waited for.
//   copies (2): the tiles' descriptors; values by tensor copies, in the swizzled
//       layout the MMA reads (V is stored token-major, which is the transposed
//       operand's contiguous side, so nothing is rearranged)
// What runs once per stream is kept out of the tile's straight line: the roles
// run different code side by side, and the instruction caches are small.
// One persistent CTA per SM; work decomposition and merge: multi_query.cuh.
//
// Measured (B200, bf16, 32 query heads over 8, head_dim 128): window of 4096 + 64
// over 32 x 8192 tokens 84 us (4.1 TB/s of the cache), 16 drafts over 8 x 8192 68 us,
// 32 drafts over 32 x 8192 300 to 318 us on different machines (430 to 460 TFLOP/s);
// the float32 kernel took 9614 us for the last. float16 at head_dim 64, the same
// window: 68 us (2.6 TB/s: a tile has half the bytes and the same chain).
// Bound by a tile's chain through the roles, foremost the softmax
// (1.15 us a tile at 16 rows, 2 us at 128, 0.5 us of which are exponentials), not by
// HBM or the tensor pipe (under 13 % active).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "multi_query.cuh"

using namespace i4kv;

namespace {

constexpr int kTile = 128, kTilePages = kTile / kMqPage;
constexpr int kDesc = 8, kSeg = 4;              // tiles, and streams, in flight between the roles
// What a stream costs besides its tiles, in tiles: its queries and its end; the
// masks of its drafts. (3 + 1 and 4 + 2 measure the same within 2 %; runs of equal
// tiles, with half the descriptor ring, took 131 instead of 118 us for 32 drafts over
// 8 x 8192 and 66 instead of 40 for 16 over 8 x 2048.)
constexpr int kStreamUnits = 2, kDraftUnits = 2;
constexpr uint64_t kTcWaitNs = 2000000000ull;   // bounded waits: 2 s
constexpr float kLazy = 14.f;                   // weights reach 2^14 (float16's range) before a rescale

// ---- tcgen05 ----
I4KV_DEVINL void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
I4KV_DEVINL void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
I4KV_DEVINL void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}
I4KV_DEVINL void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// The same with the first operand in tensor memory (two 16-bit elements a column).
I4KV_DEVINL void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// 8 columns of the warp's 32 lanes. (The waits are part of the loads' statements, so
// no use of the registers can be scheduled before them.)
I4KV_DEVINL void tc_ld8(uint32_t (&r)[8], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(addr)
      : "memory");
}
I4KV_DEVINL void tc_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
               : "memory");
}
// 16 lanes x 8 N columns in the layout of mma fragments: thread (g, t) = (lane / 4,
// lane % 4) holds columns 8 j + 2 t, + 1 of lane g in r[4 j], r[4 j + 1] and of lane
// g + 8 in r[4 j + 2], r[4 j + 3].
I4KV_DEVINL void tc_st_frag(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
I4KV_DEVINL void tc_st_frag(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
               : "memory");
}
// Two such blocks (lanes 0-15 and 16-31 of the warp's 32) and the wait for both.
I4KV_DEVINL void tc_ld_frag(uint32_t (&a)[16], uint32_t (&b)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]),
        "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(b[0]), "=r"(b[1]),
        "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]), "=r"(b[10]),
        "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15])
      : "r"(addr), "r"(addr + (16u << 16))
      : "memory");
}
I4KV_DEVINL void tc_ld_frag(uint32_t (&a)[8], uint32_t (&b)[8], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(b[0]),
        "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7])
      : "r"(addr), "r"(addr + (16u << 16))
      : "memory");
}
I4KV_DEVINL void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 4-byte asynchronous global -> shared copy.
I4KV_DEVINL void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
// One lane of a converged warp (the same one every time).
I4KV_DEVINL bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// One page of values: box of 64 channels x 16 rows x D / 64 chunks at the pool's
// page-head slab `slab` (or, of the drafts, 16 rows from `row` of head `slab`).
I4KV_DEVINL void tma_page(void* dst, const CUtensorMap* map, int row, int slab, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4}], "
      "[%5];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(slab), "r"(smem_addr(bar))
      : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle (lbo / sbo in bytes).
I4KV_DEVINL uint64_t mat_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16 with float32 accumulators; `fmt` 0
// float16, 1 bfloat16, `mn` set where both operands are contiguous along M / N.
__host__ __device__ constexpr uint32_t mma_desc(int m, int n, int fmt, bool mn) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | (mn ? (3u << 15) : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// A ring position: stage and the parity of its current use.
struct Ring {
  uint32_t s = 0, ph = 0;
  template <int N>
  I4KV_DEVINL void next() {
    if (++s == N) { s = 0; ph ^= 1; }
  }
};

template <int D, int NR>
struct Tc {
  static constexpr int CH = D / 64;                        // 64-channel chunks
  static constexpr int PAGE_V = kMqPage * D * 2;           // value bytes of a page
  static constexpr int UNIT = 16384, PPU = UNIT / PAGE_V;  // value ring: units of PPU pages
  static constexpr int NC = NR > 64 ? 64 : (NR < 32 ? NR : 32);  // rows of a softmax warpgroup
  static constexpr int WG = NR / NC, SOFT = 4 * WG;        // softmax warpgroups, warps
  static constexpr int CONV = 8;                           // two conversion groups of four warps
  static constexpr int WARPS = SOFT + CONV + 4, THREADS = 32 * WARPS;
  // Stages, as shared memory allows.
  static constexpr int NV = D == 256 ? (NR > 32 ? 4 : 5) : (NR > 64 ? 3 : (NR > 32 ? 6 : 7));  // value units
  static constexpr int NP = 2;                             // weights
  static constexpr int NB = D == 256 ? 1 : 2;              // codes and scales of a conversion group
  static_assert(NV * PPU >= kTilePages, "a whole tile's values fit (the softmax may wait for its last ones)");
  static constexpr int PC = (NR + 63) / 64;                // 64-row chunks of the weights
  static constexpr int NO = D == 256 ? 2 : 1;              // 128-channel blocks of O^T
  static constexpr int Q = NR * D * 2, P = PC * kTile * 128;
  static constexpr int KC = kTile * D / 2, SZ = kTilePages * 2 * D * 4;  // a tile's codes, and scales
  static constexpr int V_OFF = 0, Q_OFF = V_OFF + NV * UNIT, P_OFF = Q_OFF + Q, KC_OFF = P_OFF + NP * P;
  static constexpr int SZ_OFF = KC_OFF + 2 * NB * KC, END = SZ_OFF + 2 * NB * SZ;
  // Tensor memory: two tiles of S^T, O^T, two tiles of keys.
  static constexpr int COLS_O = 2 * NR, COLS_K = COLS_O + NO * NR, COLS = 512;
  static_assert(Q % 1024 == 0 && P % 1024 == 0 && COLS_K + D <= COLS, "layout");
};

struct TileDesc {
  int flags, pages, len, drafts;
  int row0, head, rows, first_row;  // rows of the sequence; the chunk's first
  int seg, slot;                // segment ring entry; record of a shared stream
  int low_edge;                 // no row sees cached positions <= low_edge (but the sinks)
  int at[kTilePages];           // position of each page's first token, -1: not there
  int slab[kTilePages];         // its page-head slab in the pools, -1: not there
  int sz[kTilePages];           // its scale slot (the first page here of its group),
  int home[kTilePages];         // and a slot's slab in the scale pool
  uint32_t slots;               // slots in use (a bit each)
  int unit;                     // units of values before it
};
enum : int { kDraftTile = 1, kMasked = 2, kFirst = 4, kLast = 8, kWhole = 16 };

template <int NR>
struct TcShared {
  uint64_t desc_full[kDesc], desc_empty[kDesc], v_full[8], v_empty[8];
  uint64_t kh_full[2], kh_empty[2], s_full[2], s_empty[2], p_full[2], p_empty[2];
  TileDesc desc[kDesc];
  uint64_t word[kSeg][kMqMaxDrafts];  // per segment: the drafts each draft sees,
  int depth[kSeg][kMqMaxDrafts];      // its ancestors,
  alignas(8) uint8_t draft[kSeg][NR];  // and each row's draft
  float qscale[kSeg][NR];       // the rows' scales,
  int qscaled[kSeg];            // where any is not 1
  int scaled[kDesc];            // the tile's keys carry scales of their own
  float kscale[kDesc][kTile];
  float ref[NR], inv[NR];       // a finished stream's references, inverse sums,
  int row[NR];                  // and rows of the outputs [rows * heads]
  alignas(8) float part[4][NR];  // maxima, or sums, over the four quarters of a tile's tokens
  unsigned long long odd[kSeg];  // per segment: drafts whose values are not all finite
  uint32_t tmem;
  RunPlan plan;
};

// Bounded wait: false (and a status bit) when its limit passes.
__device__ __noinline__ bool tc_wait_slow(uint64_t* bar, uint32_t parity, uint32_t* status) {
  if (mbar_wait_bounded(bar, parity, kTcWaitNs)) return true;
  mq_status(status, kStatusWaitTimeout);
  return false;
}
I4KV_DEVINL bool tc_wait(uint64_t* bar, uint32_t parity, uint32_t* status) {
  return mbar_try_wait(bar, parity) || tc_wait_slow(bar, parity, status);
}

template <int VK>
I4KV_DEVINL uint32_t pack16(float x, float y) {
  if constexpr (VK == INT4KV_VALUES_F16) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Two weights; float16 past its range as its largest value (bfloat16 has float32's).
template <int VK>
I4KV_DEVINL uint32_t pack_weights(float x, float y) {
  if constexpr (VK == INT4KV_VALUES_F16) {
    uint32_t w;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
    return w;
  } else {
    return pack16<VK>(x, y);
  }
}
// Two 16-bit values as float32.
template <int VK>
I4KV_DEVINL void widen2(uint32_t w, float& x, float& y) {
  if constexpr (VK == INT4KV_VALUES_F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x = f.x;
    y = f.y;
  } else {
    x = __uint_as_float(w << 16);
    y = __uint_as_float(w & 0xFFFF0000u);
  }
}

// (d0, d1) = (a0 b0 + c0, a1 b1 + c1), each rounded once.
I4KV_DEVINL void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

// 8 consecutive 16-bit inputs widened to float32.
template <int VK>
I4KV_DEVINL void widen8(const uint4& u, float (&x)[8]) {
  const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) widen2<VK>(wd[j], x[2 * j], x[2 * j + 1]);
}
template <int VK>
I4KV_DEVINL void load8(const void* base, size_t i, float (&x)[8]) {
  widen8<VK>(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i)), x);
}

// Power of two that brings |x| <= top to [1, 2) (1 for 0), and its inverse.
I4KV_DEVINL void unit_scale(float top, float& down, float& up) {
  const int e = top > 0.f ? (int)((__float_as_uint(top) >> 23) & 0xFF) : 127;
  const int c = min(max(e, 2), 252);
  down = __uint_as_float((uint32_t)(254 - c) << 23);
  up = __uint_as_float((uint32_t)c << 23);
}
// A largest magnitude in [kHalfLow, kHalfRoom) is kept as float16 unscaled.
constexpr float kHalfLow = 1.f / 256, kHalfRoom = 32768.f;
I4KV_DEVINL float finite_abs(float x) { return fabsf(x) <= 3.4e38f ? fabsf(x) : 0.f; }

// Row of the outputs [rows * heads] of a sequence's row rr, one of draft t's.
I4KV_DEVINL size_t out_row(const MultiQueryArgs& a, int row0, int head, int t, int rr) {
  return ((size_t)(row0 + t) * a.kv_heads + head) * a.group_q + (rr - t * a.group_q);
}

// ---- What runs once per stream, or rarely: kept out of the roles' loops, whose
// code has to fit the instruction caches side by side (with all of it in line the
// warps spent half of their time waiting for instructions). ----

// (They name the shared memory themselves: through a reference parameter its
// accesses would be generic ones.)
extern __shared__ __align__(1024) char tc_smem[];
template <int D, int NR>
I4KV_DEVINL TcShared<NR>& tc_shared() {
  return *reinterpret_cast<TcShared<NR>*>(tc_smem + Tc<D, NR>::END);
}

// A stream's drafts and rows, for one warp; returns the deepest draft's ancestors.
template <int D, int NR>
__device__ __noinline__ int describe_rows(const MultiQueryArgs& a, const SeqWork w, int chunk, int sg, int lane) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  uint64_t word[2] = {0, 0};
  int depth[2] = {0, 0};
  if (a.mask) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t = lane + 32 * k;
      if (t < w.drafts) {
        word[k] = (uint64_t)a.mask[w.row0 + t];
        depth[k] = draft_depth(word[k], t, w.drafts);
      }
    }
  }
  sh.depth[sg][lane] = depth[0];
  sh.depth[sg][lane + 32] = depth[1];
  if (a.mask && a.window > 0) {  // drafts behind the window are not seen either
    __syncwarp();
#pragma unroll 1
    for (int u = 0; u < w.drafts; ++u) {
      const int at = w.len + sh.depth[sg][u];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (at <= w.pos0 + depth[k] - a.window && at >= a.sinks) word[k] &= ~(1ull << u);
    }
  }
  sh.word[sg][lane] = word[0];
  sh.word[sg][lane + 32] = word[1];
#pragma unroll 1
  for (int r = lane; r < NR; r += 32) sh.draft[sg][r] = (uint8_t)(min(chunk * NR + r, w.rows - 1) / a.group_q);
  return __reduce_max_sync(0xffffffffu, max(depth[0], depth[1]));
}

// Largest finite magnitude of 8 16-bit values; and whether any exceeds float16's room.
template <int VK>
I4KV_DEVINL float top8(const uint4& u, float top) {
  float x[8];
  widen8<VK>(u, x);
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_abs(x[j]));
  return top;
}
constexpr uint32_t kBfRoom = 0x4700u, kBfLow = 0x3B80u;  // bfloat16's 2^15, 2^-8
// The bits of the largest of 8 magnitudes.
I4KV_DEVINL uint32_t top_bits(const uint4& u) {
  const uint32_t m = 0x7FFF7FFFu;
  const uint32_t t = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
  return max(t >> 16, t & 0xFFFFu);
}
// 8 16-bit values as float16; times a power of two.
template <int VK>
I4KV_DEVINL uint4 to_half8(const uint4& u) {
  if (VK == INT4KV_VALUES_F16) return u;
  float x[8];
  widen8<VK>(u, x);
  return make_uint4(pack16<INT4KV_VALUES_F16>(x[0], x[1]), pack16<INT4KV_VALUES_F16>(x[2], x[3]),
                    pack16<INT4KV_VALUES_F16>(x[4], x[5]), pack16<INT4KV_VALUES_F16>(x[6], x[7]));
}
template <int VK>
__device__ __noinline__ uint4 scale_half8(uint4 u, float down) {
  float x[8];
  widen8<VK>(u, x);
  return make_uint4(pack16<INT4KV_VALUES_F16>(x[0] * down, x[1] * down), pack16<INT4KV_VALUES_F16>(x[2] * down, x[3] * down),
                    pack16<INT4KV_VALUES_F16>(x[4] * down, x[5] * down), pack16<INT4KV_VALUES_F16>(x[6] * down, x[7] * down));
}

// Powers of two of a batch of rows' queries (bfloat16), where some row is outside
// float16's range: KT neighbouring threads hold a row.
struct Pow2 {
  float down, up;
};
template <int VK, int KT>
__device__ __noinline__ Pow2 row_scale(uint4 u, bool scaled) {
  float top = top8<VK>(u, 0.f);
#pragma unroll
  for (int o = KT / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  Pow2 p = {1.f, 1.f};
  if (scaled) unit_scale(top, p.down, p.up);
  return p;
}

// A stream's queries to shared memory, by a conversion group; D / 8 threads take a
// row together.
template <int D, int NR, int VK>
__device__ __noinline__ void load_queries(const MultiQueryArgs& a, int ds, int ct) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  constexpr int kRowThreads = D / 8, kStep = 128 / kRowThreads, kPieces = NR / kStep > 0 ? NR / kStep : 1;
  const TileDesc& d = sh.desc[ds];
  const int c8 = ct % kRowThreads, r0 = ct / kRowThreads, seg = d.seg;
  const int p16 = (c8 % 2) * 4 + (c8 % 8) / 4;  // first 16-byte piece of a row's (the next words' is 2 on)
  // channel 64 b + 16 q + 4 j + e stands at 64 b + 16 j + 4 q + e, as in the keys
  char* const to = tc_smem + Tc<D, NR>::Q_OFF + (c8 / 8) * (NR * 128) + (c8 & 2 ? 8 : 0);
  const int real = min(NR, d.rows - d.first_row);
  // row r's place: ((row0 + t) kv_heads + head) group_q + rr - t group_q, rr = first_row + r
  // (31 bits: checked on the host)
  const int place = (d.row0 * a.kv_heads + d.head) * a.group_q + d.first_row, per_draft = (a.kv_heads - 1) * a.group_q;
  const uint16_t* const q = static_cast<const uint16_t*>(a.q) + c8 * 8;
  const uint32_t mates = (kRowThreads == 32 ? 0xffffffffu : (1u << (kRowThreads & 31)) - 1) << (ct % 32 / kRowThreads * kRowThreads);
  constexpr int kBatch = kPieces < 8 ? kPieces : 8;  // loads in flight
  static_assert(kStep <= NR, "every thread has a row");
#pragma unroll 1
  for (int k0 = 0; k0 < kPieces; k0 += kBatch) {
    uint4 u[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = r0 + (k0 + k) * kStep;
      u[k] = make_uint4(0, 0, 0, 0);
      if (r < real)
        u[k] = __ldg(reinterpret_cast<const uint4*>(q + (size_t)(place + r + sh.draft[seg][r] * per_draft) * D));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = r0 + (k0 + k) * kStep;
      uint4 h = to_half8<VK>(u[k]);
      if (VK == INT4KV_VALUES_BF16) {
        const uint32_t top = top_bits(u[k]);
        const uint32_t high = __ballot_sync(0xffffffffu, top >= kBfRoom), some = __ballot_sync(0xffffffffu, top >= kBfLow);
        const bool scaled = r < real && ((high & mates) || !(some & mates));
        float up = 1.f;
        if (__any_sync(0xffffffffu, scaled)) {
          const Pow2 p = row_scale<VK, kRowThreads>(u[k], scaled);
          if (scaled) h = scale_half8<VK>(u[k], p.down);
          up = p.up;
          if (up != 1.f) sh.qscaled[seg] = 1;
        }
        if (c8 == 0) sh.qscale[seg][r] = up;
      }
      char* at = to + r * 128;
      *reinterpret_cast<uint2*>(at + ((p16 ^ (r & 7)) << 4)) = make_uint2(h.x, h.y);
      *reinterpret_cast<uint2*>(at + (((p16 + 2) ^ (r & 7)) << 4)) = make_uint2(h.z, h.w);
    }
  }
  fence_proxy_async_smem();
}

// Keys, by a conversion group: thread (g, t) of a warp takes tokens g, g + 8 of each
// of the warp's two pages and 16 channels 64 b + 16 t of each block b of 64: its
// parameters stay in registers over the tokens, and the fragments go to tensor
// memory as they are. Rows of codes are swizzled by 16 bytes, as the threads of a
// warp read 8 rows at a time.
template <int D>
I4KV_DEVINL int code_swizzle(int t) {
  return D == 64 ? (t >> 2 & 1) : (D == 128 ? (t >> 1 & 3) : (t & 7));
}
template <int D, bool SCALED>
I4KV_DEVINL void convert_keys(const TileDesc& d, const char* codes, const float* scales, uint32_t keys, int ct, float down_a,
                              float down_b) {
  const int lane = ct & 31, g = lane >> 2, t4 = lane & 3, page0 = (ct >> 5) * 2;
  const int slot_a = d.sz[page0], slot_b = d.sz[page0 + 1];  // (uniform in the warp)
#pragma unroll 1
  for (int blk = 0; blk < D / 64; ++blk) {
    float e[16], z[16];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (p == 0 || slot_b != slot_a || SCALED) {
        const float* sz = scales + (p ? slot_b : slot_a) * (2 * D) + 64 * blk + 16 * t4;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 x = *reinterpret_cast<const float4*>(sz + j);
          const float4 y = *reinterpret_cast<const float4*>(sz + D + j);
          e[j] = x.x; e[j + 1] = x.y; e[j + 2] = x.z; e[j + 3] = x.w;
          z[j] = y.x; z[j + 1] = y.y; z[j + 2] = y.z; z[j + 3] = y.w;
        }
        if constexpr (SCALED) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            e[j] *= p ? down_b : down_a;
            z[j] *= p ? down_b : down_a;
          }
        }
      }
      uint32_t h[16];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int t = (page0 + p) * kMqPage + g + 8 * r;
        // 16 channels: 8 bytes, half of the row's 16-byte piece 2 blk + t4 / 2
        const uint2 wd = *reinterpret_cast<const uint2*>(codes + t * (D / 2) + 8 * (t4 & 1) +
                                                         (((2 * blk + (t4 >> 1)) ^ code_swizzle<D>(t)) << 4));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t w4 = k ? wd.y : wd.x;
          const uint32_t lo = (w4 & 0x0F0F0F0Fu) | 0x80808080u, hi = ((w4 >> 4) & 0x0F0F0F0Fu) | 0x80808080u;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = 8 * k + 2 * j;
            float x0, x1;
            fma2(x0, x1, __uint_as_float(__byte_perm(lo, 0x3F000000u, 0x7044u | (j << 8))),
                 __uint_as_float(__byte_perm(hi, 0x3F000000u, 0x7044u | (j << 8))), e[c], e[c + 1], z[c], z[c + 1]);
            h[4 * (2 * k + j / 2) + 2 * r + j % 2] = pack16<INT4KV_VALUES_F16>(x0, x1);
          }
        }
      }
      tc_st_frag(keys + ((uint32_t)(16 * p) << 16) + 32 * blk, h);
    }
  }
}

// The same with a power of two per group, for keys outside float16's range.
template <int D, int NR>
__device__ __noinline__ void convert_scaled(int ds, const char* codes, const float* scales, uint32_t keys, int ct) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  const TileDesc& d = sh.desc[ds];
  const int lane = ct & 31, page0 = (ct >> 5) * 2;
  float down[2];
#pragma unroll 1
  for (int p = 0; p < 2; ++p) {
    const float* sz = scales + d.sz[page0 + p] * (2 * D);
    float top = 0.f, dn, up;
#pragma unroll 1
    for (int ch = lane; ch < D; ch += 32) {
      const float e = sz[ch], z = sz[D + ch];  // code 0: e + z; 15: 143/128 e + z
      top = fmaxf(top, fmaxf(finite_abs(e + z), finite_abs(fmaf(143.f / 128.f, e, z))));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    unit_scale(top, dn, up);
    if (p == 0) down[0] = dn; else down[1] = dn;
    if (lane < kMqPage) sh.kscale[ds][(page0 + p) * kMqPage + lane] = up;
  }
  convert_keys<D, true>(d, codes, scales, keys, ct, down[0], down[1]);
}

// Drafted keys, as they are, or (true) with a power of two each where one of them
// (or a thread's share of it) is outside float16's range.
template <int D, int NR, int VK>
__device__ __noinline__ bool draft_keys(const MultiQueryArgs& a, int ds, uint32_t keys, int ct, int bar) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  const TileDesc& d = sh.desc[ds];
  const int lane = ct & 31, g = lane >> 2, t4 = lane & 3, page0 = (ct >> 5) * 2, drafts = d.drafts, pages = d.pages;
  const uint16_t* const base = static_cast<const uint16_t*>(a.kd) + ((size_t)d.row0 * a.kv_heads + d.head) * D + 16 * t4;
  const size_t step = (size_t)a.kv_heads * D;
  bool scaled = false;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    uint32_t big = 0;
#pragma unroll 1
    for (int p = 0; p < 2; ++p) {
      if (page0 + p >= pages) break;  // (nothing there is seen)
      const int ta = (page0 + p) * kMqPage + g, tb = ta + 8;
      const uint16_t *sa = base + ta * step, *sb = base + tb * step;
      float down[2] = {1.f, 1.f};
      if (scaled) {
#pragma unroll 1
        for (int r = 0; r < 2; ++r) {
          float top = 0.f, up, dn;
#pragma unroll 1
          for (int blk = 0; blk < D / 64; ++blk)
#pragma unroll 1
            for (int e = 0; e < 2; ++e)
              if ((r ? tb : ta) < drafts)
                top = top8<VK>(__ldg(reinterpret_cast<const uint4*>((r ? sb : sa) + 64 * blk + 8 * e)), top);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          unit_scale(top, dn, up);
          if (r) down[1] = dn; else down[0] = dn;
          if (t4 == 0) sh.kscale[ds][r ? tb : ta] = up;
        }
      }
      uint32_t top[2] = {0, 0};
#pragma unroll 1
      for (int blk = 0; blk < D / 64; ++blk) {
        uint4 u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // token k / 2, half k % 2 of the channels
          u[k] = make_uint4(0, 0, 0, 0);
          if ((k / 2 ? tb : ta) < drafts)
            u[k] = __ldg(reinterpret_cast<const uint4*>((k / 2 ? sb : sa) + 64 * blk + 8 * (k % 2)));
        }
        uint32_t h[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          top[k / 2] = max(top[k / 2], top_bits(u[k]));
          uint4 v = to_half8<VK>(u[k]);
          if (scaled) v = scale_half8<VK>(u[k], down[k / 2]);
          // channels 8 e + 2 j, + 1: fragment column (2 e + j / 2), word j % 2
          h[8 * (k % 2) + 2 * (k / 2)] = v.x;
          h[8 * (k % 2) + 2 * (k / 2) + 1] = v.y;
          h[8 * (k % 2) + 4 + 2 * (k / 2)] = v.z;
          h[8 * (k % 2) + 4 + 2 * (k / 2) + 1] = v.w;
        }
        __syncwarp();
        tc_st_frag(keys + ((uint32_t)(16 * p) << 16) + 32 * blk, h);
      }
      big |= (ta < drafts && (top[0] < kBfLow || top[0] >= kBfRoom)) || (tb < drafts && (top[1] < kBfLow || top[1] >= kBfRoom));
    }
    if (VK == INT4KV_VALUES_F16 || scaled || !named_bar_or(bar, 128, big)) break;
    scaled = true;
  }
  return scaled;
}

// Whether some row sees the token `at` of a tile at all (a cached one).
I4KV_DEVINL bool token_real(const MultiQueryArgs& a, const TileDesc& d, int page, int at) {
  const bool draft = d.flags & kDraftTile;
  const bool here = page < d.pages && d.at[page] >= 0 && at < (draft ? d.drafts : d.len);
  return here && (draft || a.window == 0 || at > d.low_edge || at < a.sinks);
}

// Logits of scaled keys or queries, brought back in tensor memory, so nothing else
// has to know. A thread takes one token. (What is not there is masked afterwards.)
template <int D, int NR>
__device__ __noinline__ void scale_tile(int ds, uint32_t s_addr, int c0, int tok) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  const int sg = sh.desc[ds].seg;
  const float ks = sh.scaled[ds] ? sh.kscale[ds][tok] : 1.f;
  const bool rows = sh.qscaled[sg];
#pragma unroll 1
  for (int j0 = 0; j0 < Tc<D, NR>::NC; j0 += 8) {
    uint32_t x[8];
    tc_ld8(x, s_addr + j0);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = __float_as_uint(__uint_as_float(x[j]) * (ks * (rows ? sh.qscale[sg][c0 + j0 + j] : 1.f)));
    __syncwarp();
    tc_st8(s_addr + j0, x);
  }
  tc_wait_st();
}

// A tile that some row does not see all of: the logits it must not see become -inf
// in tensor memory, so nothing else has to know. A thread takes one token; whether
// row r sees it hangs on the row's draft, the same for the whole warp.
template <int D, int NR>
__device__ __noinline__ void mask_tile(const MultiQueryArgs& a, int ds, uint32_t s_addr, int c0, int tok) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  const TileDesc& d = sh.desc[ds];
  const int sg = d.seg, page = tok / kMqPage, at = d.at[page] + tok % kMqPage;
  const bool draft = d.flags & kDraftTile, real = token_real(a, d, page, at);
  // the drafts that see the token: of the cached ones all, but for the window's edge
  uint32_t seen[2] = {0, 0};
  if (real) {
    const bool edge = !draft && a.window > 0 && at >= a.sinks;
    if (draft || edge) {
      const int drafts = max(1, d.drafts);  // (a window's one query counts as draft 0)
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        uint32_t s = 0;
#pragma unroll 4
        for (int t = 0; t < min(32, drafts - 32 * h); ++t)
          s |= (uint32_t)(draft ? sh.word[sg][32 * h + t] >> (at & 63) & 1 : at > d.low_edge + sh.depth[sg][32 * h + t]) << t;
        if (h) seen[1] = s; else seen[0] = s;
      }
    } else {
      seen[0] = seen[1] = 0xFFFFFFFFu;
    }
  }
#pragma unroll 1
  for (int j0 = 0; j0 < Tc<D, NR>::NC; j0 += 8) {
    uint32_t x[8];
    tc_ld8(x, s_addr + j0);
    const uint2 rows = *reinterpret_cast<const uint2*>(&sh.draft[sg][c0 + j0]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = (j < 4 ? rows.x >> (8 * j) : rows.y >> (8 * j - 32)) & 63;
      if (!((t < 32 ? seen[0] : seen[1]) >> (t & 31) & 1)) x[j] = 0xFF800000u;
    }
    __syncwarp();
    tc_st8(s_addr + j0, x);
  }
  tc_wait_st();
}

// A softmax thread's rows: minus the references, and the sums.
template <int NI>
struct RowState {
  float nref[NI][2], l[NI][2];
  bool failed;
};
// The reference of a row that has seen nothing: below every logit but those the factor
// log2 e takes to (minus) infinity.
constexpr float kNoRef = -3e38f;

// Raise the references to the true maxima of the tile, rescale sums and outputs. A
// weight is 2^(x log2 e - ref), the product unrounded, so the references are rounded
// down: a row's largest weight is then 1 or more whatever the logits' size (rounded to
// nearest it came below float16's smallest for logits past 2^27). What it is above 1,
// less than 2^(2^-23 |ref|), float16 cuts at its largest value; logits that large are
// too far apart for a second one to come near.
// `prev`: the buffer of the last tile's weights (-1: O^T holds nothing yet).
template <int D, int NR>
__device__ __noinline__ RowState<Tc<D, NR>::NC / 8> raise_references(const MultiQueryArgs& a, RowState<Tc<D, NR>::NC / 8> s,
                                                                     uint32_t s_addr, uint32_t o_addr, int c0,
                                                                     int quarter, int lane, int prev, uint32_t parity,
                                                                     int bar) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  using T = Tc<D, NR>;
  constexpr int NI = T::NC / 8, LI = NI < 4 ? NI : 4;
  const int g = lane >> 2, t4 = lane & 3;
  // Maxima of 2 NI rows over a thread's four tokens, then over the 8 threads with the
  // same t4: each gives half of its rows away and keeps the other, three times.
  float m[2 * NI];
#pragma unroll
  for (int j0 = 0; j0 < NI; j0 += LI) {
    uint32_t x[2][4 * LI];
    tc_ld_frag(x[0], x[1], s_addr + 8 * j0);
#pragma unroll
    for (int j = 0; j < LI; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        m[2 * (j0 + j) + e] = fmaxf(fmaxf(__uint_as_float(x[0][4 * j + e]), __uint_as_float(x[0][4 * j + 2 + e])),
                                    fmaxf(__uint_as_float(x[1][4 * j + e]), __uint_as_float(x[1][4 * j + 2 + e])));
    }
  }
  int at = 0;  // first of the pairs of rows this thread keeps
#pragma unroll
  for (int o = 4, n = 2 * NI; o > 0; o >>= 1) {
    if (n > 2) {  // (pairs stay together)
      n /= 2;
      const bool upper = g & o;
      at += upper ? n / 2 : 0;
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const float give = upper ? m[k] : m[k + n], keep = upper ? m[k + n] : m[k];
        m[k] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, 4 * o));
      }
    } else {
      m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], 4 * o));
      m[1] = fmaxf(m[1], __shfl_xor_sync(0xffffffffu, m[1], 4 * o));
    }
  }
  *reinterpret_cast<float2*>(&sh.part[quarter][c0 + 8 * at + 2 * t4]) =
      make_float2(fmaxf(__fmul_rd(m[0], kLog2e), kNoRef), fmaxf(__fmul_rd(m[1], kLog2e), kNoRef));
  s.failed = prev >= 0 && !tc_wait(&sh.p_empty[prev & 1], parity, a.status);  // the weights of tile i - 1 have been multiplied
  named_bar_sync(bar, 128);
  tc_fence_after();
#pragma unroll
  for (int j0 = 0; j0 < NI; j0 += LI) {
    float al[LI][2];
#pragma unroll
    for (int j = 0; j < LI; ++j) {
      float2 top = make_float2(-s.nref[j0 + j][0], -s.nref[j0 + j][1]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 p = *reinterpret_cast<const float2*>(&sh.part[q][c0 + 8 * (j0 + j) + 2 * t4]);
        top = make_float2(fmaxf(top.x, p.x), fmaxf(top.y, p.y));
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float m = e ? top.y : top.x;
        al[j][e] = exp2_fast(-s.nref[j0 + j][e] - m);
        s.nref[j0 + j][e] = -m;
        s.l[j0 + j][e] *= al[j][e];
      }
    }
    if (prev >= 0) {
#pragma unroll 1
      for (int o = 0; o < T::NO; ++o) {
        const uint32_t at_o = o_addr + o * NR + 8 * j0;
        uint32_t x[2][4 * LI];
        tc_ld_frag(x[0], x[1], at_o);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int k = 0; k < 4 * LI; ++k) x[q][k] = __float_as_uint(__uint_as_float(x[q][k]) * al[k / 4][k % 2]);
          tc_st_frag(at_o + ((uint32_t)(16 * q) << 16), x[q]);
        }
      }
    }
  }
  if (prev >= 0) {
    tc_wait_st();
    tc_fence_before();
  }
  return s;
}

// Values that no row sees must not reach the product (0 * NaN): cleared. A drafted
// value that is not finite is taken out too and added for the rows that see it when
// the stream ends. One thread a token. (The values of tile i - 1 have been multiplied
// before those of tile i are waited for: a short ring reuses their units, and a wait
// tells a phase from its neighbours only.)
template <int D, int NR, int VK>
__device__ __noinline__ bool clear_values(const MultiQueryArgs& a, int ds, int i, int tok) {
  using T = Tc<D, NR>;
  TcShared<NR>& sh = tc_shared<D, NR>();
  const TileDesc& d = sh.desc[ds];
  bool ok = true;
  const int at = d.at[tok / kMqPage] + tok % kMqPage;
  const bool draft = d.flags & kDraftTile, real = token_real(a, d, tok / kMqPage, at);
  if (tok < d.pages * kMqPage && (!real || draft)) {
    const int u = d.unit + tok / (kMqPage * T::PPU), s = u % T::NV;
    ok = (i == 0 || tc_wait(&sh.p_empty[(i - 1) % T::NP], ((i - 1) / T::NP) & 1, a.status)) &&
         tc_wait(&sh.v_full[s], (u / T::NV) & 1, a.status);
    char* row = tc_smem + T::V_OFF + s * T::UNIT + (tok / kMqPage % T::PPU) * T::PAGE_V + (tok % kMqPage) * 128;
    // (the order of a thread's 16-byte pieces spreads a warp's over the banks)
    auto piece = [&](int q) {
      return reinterpret_cast<uint4*>(row + (q / 8) * (kMqPage * 128) + 16 * (q % 8 ^ (tok & 7)));
    };
    bool bad = false;
    if (!real) {
#pragma unroll 4
      for (int q = 0; q < 8 * T::CH; ++q) *piece(q) = make_uint4(0, 0, 0, 0);
    } else {
      // an exponent of all ones carries into the sign's place
      constexpr uint32_t kExp = VK == INT4KV_VALUES_F16 ? 0x7C007C00u : 0x7F807F80u;
      constexpr uint32_t kOne = VK == INT4KV_VALUES_F16 ? 0x04000400u : 0x00800080u;
      uint32_t any = 0;
#pragma unroll 4
      for (int q = 0; q < 8 * T::CH; ++q) {
        const uint4 y = *piece(q);
        any |= ((y.x & kExp) + kOne) | ((y.y & kExp) + kOne) | ((y.z & kExp) + kOne) | ((y.w & kExp) + kOne);
      }
      bad = any & 0x80008000u;
      if (bad) {
#pragma unroll 1
        for (int q = 0; q < 32 * T::CH; ++q) {
          uint32_t* y = reinterpret_cast<uint32_t*>(piece(q / 4)) + q % 4;
          const uint32_t m = ((*y & kExp) + kOne) & 0x80008000u;
          if (m) *y &= (m & 0x8000u ? 0u : 0x0000FFFFu) | (m >> 31 ? 0u : 0xFFFF0000u);
        }
      }
    }
    if (bad) atomicOr(&sh.odd[d.seg], 1ull << (at & 63));
  }
  __syncwarp();
  return ok;
}

// Drafted values that are not finite, for the rows that see them (8 rows from `col`).
struct Eight {
  uint32_t x[8];
};
template <int D, int NR, int VK>
__device__ __noinline__ Eight add_odd_values(const MultiQueryArgs& a, int ds, unsigned long long odd, int ch, int col,
                                             Eight e) {
  TcShared<NR>& sh = tc_shared<D, NR>();
  const TileDesc& d = sh.desc[ds];
#pragma unroll 1
  for (unsigned long long left = odd; left; left &= left - 1) {
    const int u = __ffsll(left) - 1;
    float y2[2];
    load_f32<2>(a.vd, VK, ((size_t)(d.row0 + u) * a.kv_heads + d.head) * D + (ch & ~1), y2);
    const float y = ch & 1 ? y2[1] : y2[0];
    if (fabsf(y) <= 3.4e38f) continue;
#pragma unroll 1
    for (int j = 0; j < 8; ++j)
      if (sh.word[d.seg][sh.draft[d.seg][col + j]] >> u & 1) e.x[j] = __float_as_uint(__uint_as_float(e.x[j]) + y);
  }
  __syncwarp();
  return e;
}

// A stream's (or a run's share of it) end, by one softmax warpgroup: the sums of its
// warps are in sh.part, its products are done. O^T, a lane a channel, over the sums,
// or as a record.
template <int D, int NR, int VK>
__device__ __noinline__ void finish_stream(const MultiQueryArgs& a, int ds, uint32_t tm, int c0, int tok, int bar) {
  using T = Tc<D, NR>;
  TcShared<NR>& sh = tc_shared<D, NR>();
  const TileDesc& d = sh.desc[ds];
  const bool whole = d.flags & kWhole;
  const int sg = d.seg;
  float* rec = a.recs + (size_t)d.slot * Record<NR, D>::kFloats;
  if (tok < T::NC) {
    const int r = c0 + tok, rr = d.first_row + r;
    const float sum = (sh.part[0][r] + sh.part[1][r]) + (sh.part[2][r] + sh.part[3][r]);
    sh.inv[r] = 1.f / fmaxf(sum, 1e-10f);
    sh.row[r] = (int)out_row(a, d.row0, d.head, sh.draft[sg][r], rr);
    if (!whole) {
      rec[r] = sh.ref[r] == kNoRef ? -INFINITY : sh.ref[r] * 0.6931471805599453f;
      rec[NR + r] = sum;
    }
  }
  named_bar_sync(bar, 128);
  tc_fence_after();
  const unsigned long long odd = sh.odd[sg];
  const int cols = min(T::NC, d.rows - d.first_row - c0);  // rows that are there
#pragma unroll 1
  for (int o = 0; o < T::NO; ++o) {
    const int ch = o * 128 + tok;
    if (o * 128 + (tok & 96) >= D) break;  // (a warp's channels are all there or none is)
#pragma unroll 1
    for (int j0 = 0; j0 < cols; j0 += 8) {
      const int col = c0 + j0;
      uint32_t x[8];
      tc_ld8(x, tm + T::COLS_O + o * NR + col);
      if (odd) {
        Eight e;
#pragma unroll
        for (int j = 0; j < 8; ++j) e.x[j] = x[j];
        e = add_odd_values<D, NR, VK>(a, ds, odd, ch, col, e);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = e.x[j];
      }
      if (whole) {
        const float4 i0 = *reinterpret_cast<const float4*>(&sh.inv[col]), i1 = *reinterpret_cast<const float4*>(&sh.inv[col + 4]);
        const int4 r0 = *reinterpret_cast<const int4*>(&sh.row[col]), r1 = *reinterpret_cast<const int4*>(&sh.row[col + 4]);
        const float inv[8] = {i0.x, i0.y, i0.z, i0.w, i1.x, i1.y, i1.z, i1.w};
        const int row[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j0 + j >= cols) break;
          const float y = __uint_as_float(x[j]) * inv[j];
          const size_t to = (size_t)row[j] * D + ch;
          if constexpr (VK == INT4KV_VALUES_F16) static_cast<__half*>(a.out)[to] = __float2half_rn(y);
          else static_cast<__nv_bfloat16*>(a.out)[to] = __float2bfloat16_rn(y);
        }
      } else {
        float* to = rec + 2 * NR + (size_t)col * D + ch;
#pragma unroll
        for (int j = 0; j < 8; ++j) to[j * D] = __uint_as_float(x[j]);
      }
    }
  }
  tc_fence_before();
  __syncwarp();
}

template <int D, int NR, int VK>
__global__ void __launch_bounds__(Tc<D, NR>::THREADS, 1)
multi_query_tc_kernel(const __grid_constant__ MultiQueryArgs a, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ CUtensorMap dmap) {
  using T = Tc<D, NR>;
  constexpr int kSoftWarps = T::SOFT, kConvWarps = T::CONV;
  constexpr int kMmaWarp = kSoftWarps + kConvWarps, kOutWarp = kMmaWarp + 1, kCopyWarp = kMmaWarp + 2;  // two copy warps
  constexpr int kBarConv = 1, kBarGroup = 3;  // named barriers: one per conversion group, one per softmax warpgroup
  char* const smem = tc_smem;  // (no static shared memory: it starts on a 1024-byte boundary)
  TcShared<NR>& sh = tc_shared<D, NR>();
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)),
                 "n"(T::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  if (tid == 0) {
    for (int i = 0; i < kDesc; ++i) {
      mbar_init(&sh.desc_full[i], 1);
      mbar_init(&sh.desc_empty[i], kSoftWarps + 4 + 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.kh_full[i], 4);
      mbar_init(&sh.kh_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_empty[i], kSoftWarps);
      mbar_init(&sh.p_full[i], kSoftWarps);
      mbar_init(&sh.p_empty[i], 1);
    }
    for (int i = 0; i < 8; ++i) {
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 1);
    }
    fence_barrier_init();
  }
  grid_dependency_wait();
  allow_dependent_launch();
  if (!a.offs) zero_idle_rows<NR, kTilePages, D>(a);
  const int cta = blockIdx.x;
  if (warp == kCopyWarp) {
    const RunPlan mine = plan_run<NR, kTilePages, kStreamUnits, kDraftUnits>(a, cta, gridDim.x);
    if (lane == 0) {
      sh.plan = mine;
      // (the same thread writes the note of the run's last tile, which a wait that runs out
      // keeps it from: until then, and then for good, this run shares no stream)
      a.tails[cta] = RunTail{};
    }
  }
  __syncthreads();
  tc_fence_after();
  const int n_tiles = sh.plan.tiles;
  const uint32_t tm = sh.tmem;

  if (n_tiles == 0) {
  } else if (warp >= kCopyWarp) {
    // ------------------------------------------------------------ copies
    // Both warps walk the tiles; the first publishes their descriptors, the second
    // copies the values.
    const bool values = warp > kCopyWarp;
    const RunPlan plan = sh.plan;
    SeqWork w = seq_work<NR, kTilePages>(a, plan.b, false);
    TileAt p = tile_at(a, w, plan.b, plan.rem);
    int seg = -1, high_edge = 0;
    int end1 = -1, end2 = -1, end3 = -1;  // last tiles of the streams before the last one, ..
    Ring v;
    bool ok = true;
    // Lane 8 k + j: page j of tile set + k (and the page its scales are kept with),
    // and of the four tiles behind those, loaded while these four are in work.
    static_assert(kTilePages == 8, "four tiles a warp");
    int set = 0, phys4 = -1, home4 = -1, phys_next = -1, home_next = -1;
    auto load_set = [&](int tile, int& ph, int& hm) {
      ph = hm = -1;
      tile += lane >> 3;
      const int pg = tile_page<kTilePages>(w, tile, lane & 7);
      if (tile < w.cache_tiles && page_visible(w, pg)) {
        const int32_t* bt = a.block_table + (size_t)p.b * a.max_pages;
        ph = __ldg(bt + pg);
        hm = __ldg(bt + pg / a.group_pages * a.group_pages);
      }
    };
    bool turn = true;  // a new stream
    int units = 0;
#pragma unroll 1
    for (int i = 0; i < n_tiles && ok; ++i) {
      const int ds = i % kDesc;
      const bool draft = p.tile >= w.cache_tiles;
      if (turn || p.tile == set + 4) {
        set = p.tile;
        phys4 = phys_next;
        home4 = home_next;
        if (turn) load_set(set, phys4, home4);
        load_set(set + 4, phys_next, home_next);
        turn = false;
      }
      const int from = 8 * (p.tile - set) + (lane & 7), pg = tile_page<kTilePages>(w, p.tile, lane & 7);
      const int phys = __shfl_sync(0xffffffffu, phys4, from);
      int home = __shfl_sync(0xffffffffu, home4, from);
      const int here = draft ? (w.drafts + kMqPage - 1) / kMqPage
                             : min(kTilePages, w.pages - tile_page<kTilePages>(w, p.tile, 0));
      const bool mine = lane < here && (draft || page_visible(w, pg));
      const bool live = mine && (draft || (phys >= 0 && phys < a.num_pages && home >= 0 && home < a.num_pages));
      const uint32_t lives = __ballot_sync(0xffffffffu, live);
      if (!values) {
        ok = __all_sync(0xffffffffu, tc_wait(&sh.desc_empty[ds], (i / kDesc + 1) & 1, a.status));
        if (!ok) break;
        const bool first = i == 0 || p.tile == 0;
        if (first) {
          // (the stream kSeg before this one has left its ring entry)
          if (++seg >= kSeg && end3 > i - kDesc)
            ok = __all_sync(0xffffffffu, tc_wait(&sh.desc_empty[end3 % kDesc], (end3 / kDesc) & 1, a.status));
          if (!ok) break;
          end3 = end2;
          end2 = end1;
          end1 = i - 1;
          high_edge = w.pos0 + describe_rows<D, NR>(a, w, p.chunk, seg % kSeg, lane) - a.window;
        }
        int at = -1;
        bool clean = lane >= here;  // every row sees all of the page
        if (mine) {
          if (draft) {
            at = lane * kMqPage;
          } else {
            if (!live) mq_status(a.status, kStatusBadPage);
            at = live ? pg * kMqPage : -1;
            clean = live && at + kMqPage <= w.len &&
                    (a.window == 0 || at > high_edge || at + kMqPage <= a.sinks);
          }
        }
        const bool masked = !__all_sync(0xffffffffu, clean) || here < kTilePages;
        // pages of one group share a scale slot: the slot of the group's first page here
        if (!live) home = -1;
        const int prev = __shfl_up_sync(0xffffffffu, home, 1);
        const uint32_t starts = __ballot_sync(0xffffffffu, live && (lane == 0 || home != prev));
        if (lane < kTilePages) {
          TileDesc& d = sh.desc[ds];
          d.at[lane] = at;
          d.slab[lane] = live && !draft ? phys * a.kv_heads + p.head : -1;
          d.home[lane] = live && !draft ? home * a.kv_heads + p.head : -1;
          d.sz[lane] = max(0, 31 - __clz(starts & ((2u << lane) - 1)));
        }
        if (lane == 0) {
          TileDesc& d = sh.desc[ds];
          const int first_u = i - p.tile;  // the stream's first tile, of the run's
          const bool ends = p.tile + 1 == w.tiles;
          d.flags = (draft ? kDraftTile : 0) | (masked ? kMasked : 0) | (first ? kFirst : 0) |
                    ((ends || i + 1 == n_tiles) ? kLast : 0) | ((ends && first_u >= 0) ? kWhole : 0);
          d.pages = here;
          d.len = w.len;
          d.drafts = w.drafts;
          d.row0 = w.row0;
          d.head = p.head;
          d.rows = w.rows;
          d.first_row = p.chunk * NR;
          d.seg = seg % kSeg;
          d.slot = 2 * cta + (first_u > 0 ? 1 : 0);
          d.low_edge = a.window > 0 ? w.pos0 - a.window : -1;
          d.slots = draft ? 0 : starts;
          d.unit = units;
          if (first) sh.odd[seg % kSeg] = sh.qscaled[seg % kSeg] = 0;
          if (i + 1 == n_tiles) note_tail(a, cta, plan, w, p, NR);
        }
        units += (here + T::PPU - 1) / T::PPU;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.desc_full[ds]);
      } else {
        const CUtensorMap* map = draft ? &dmap : &vmap;
        const int row = draft ? w.row0 + lane * kMqPage : 0, slab = draft ? p.head : phys * a.kv_heads + p.head;
#pragma unroll 1
        for (int g0 = 0; g0 < here; g0 += T::PPU) {
          ok = ok && tc_wait(&sh.v_empty[v.s], v.ph ^ 1, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint64_t* bar = &sh.v_full[v.s];
          const uint32_t unit = lives >> g0 & ((1u << T::PPU) - 1);
          char* dst = smem + T::V_OFF + v.s * T::UNIT;
          if (elect_one()) mbar_arrive_expect_tx(bar, __popc(unit) * T::PAGE_V);
          __syncwarp();
          if (lane >= g0 && lane < g0 + T::PPU && live) tma_page(dst + (lane - g0) * T::PAGE_V, map, row, slab, bar);
          __syncwarp();
          v.next<T::NV>();
        }
        if (!ok) break;
      }
      if (++p.tile >= w.tiles) {
        next_stream<NR, kTilePages>(a, w, p);
        turn = true;
      }
    }
    // after a timeout: the copies issued so far land (or a bound passes) before the CTA ends
    if (!ok && lane == 0) {
      for (int s = 0; s < T::NV && values; ++s) mbar_wait_bounded(&sh.v_full[s], s < (int)v.s ? v.ph : v.ph ^ 1, 10000000ull);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ S^T = K^ Q^T
    constexpr uint32_t kQk = mma_desc(128, NR, 0, false);
    const uint32_t base = smem_addr(smem);
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
      const int hb = i & 1;
      ok = tc_wait(&sh.kh_full[hb], (i / 2) & 1, a.status) && tc_wait(&sh.s_empty[hb], (i / 2 + 1) & 1, a.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t keys = tm + T::COLS_K + hb * (D / 2);
        const uint64_t qd = mat_desc(base + T::Q_OFF, 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma_ts(tm + hb * NR, keys + k * 8, qd + (k / 4) * (NR * 128 / 16) + (k % 4) * 2, kQk, k > 0);
        tc_commit(&sh.s_full[hb]);
        tc_commit(&sh.kh_empty[hb]);
      }
      __syncwarp();
    }
  } else if (warp == kOutWarp) {
    // ------------------------------------------------------------ O^T += V^T P^T
    constexpr uint32_t kPv = mma_desc(128, NR, VK == INT4KV_VALUES_BF16 ? 1 : 0, true);
    const uint32_t base = smem_addr(smem);
    Ring v;
#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
      const int ds = i % kDesc, pb = i % T::NP;
      bool ok = tc_wait(&sh.desc_full[ds], (i / kDesc) & 1, a.status);
      const int pages = ok ? sh.desc[ds].pages : 0;
      const bool fresh = sh.desc[ds].flags & kFirst;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.desc_empty[ds]);
      ok = ok && tc_wait(&sh.p_full[pb], (i / T::NP) & 1, a.status);
      const uint64_t pd = mat_desc(base + T::P_OFF + pb * T::P, kTile * 128, 1024);
#pragma unroll 1
      for (int g0 = 0; g0 < pages; g0 += T::PPU) {
        ok = ok && tc_wait(&sh.v_full[v.s], v.ph, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = mat_desc(base + T::V_OFF + v.s * T::UNIT, 2048, 1024);
#pragma unroll
          for (int q = 0; q < T::PPU; ++q) {
            if (g0 + q < pages) {
#pragma unroll
              for (int o = 0; o < T::NO; ++o)  // (head_dim 64: lanes 64-127 take what follows, and are not read)
                tc_mma(tm + T::COLS_O + o * NR, vd + (q * T::PAGE_V + o * 4096) / 16, pd + (g0 + q) * (2048 / 16), kPv,
                       !(fresh && g0 + q == 0));
            }
          }
          tc_commit(&sh.v_empty[v.s]);
          if (g0 + T::PPU >= pages) tc_commit(&sh.p_empty[pb]);
        }
        __syncwarp();
        v.next<T::NV>();
      }
      if (!__all_sync(0xffffffffu, ok)) break;
    }
  } else if (warp >= kSoftWarps) {
    // ------------------------------------------------------------ conversion
    const int grp = (warp - kSoftWarps) / 4, ct = (warp - kSoftWarps) % 4 * 32 + lane;
    const int bar = kBarConv + grp;
    // (a warp reaches the lanes of tensor memory that its number within the
    // warpgroup names: kSoftWarps is a multiple of 4)
    const uint32_t lanes = (uint32_t)(ct & 96) << 16;
    // A tile's codes and scales are copied ahead into one of two buffers; a thread
    // turns the scales it copied into what the conversion uses, and the group meets
    // once before it reads either. (The other buffer is free by then: every warp
    // has left the tile that used it. With one buffer, at head_dim 256, the group
    // meets again before the next copies.) Rows of codes are swizzled by 16 bytes, as
    // the threads of a warp read 8 rows at a time.
    constexpr int kRow = D / 2;  // bytes of a row of codes
    auto codes_of = [&](int i) { return smem + T::KC_OFF + (T::NB * grp + (i >> 1 & (T::NB - 1))) * T::KC; };
    auto scales_of = [&](int i) {
      return reinterpret_cast<float*>(smem + T::SZ_OFF + (T::NB * grp + (i >> 1 & (T::NB - 1))) * T::SZ);
    };
    auto prefetch = [&](const TileDesc& d, int i) {
      const int slab = d.slab[ct / kMqPage];
      if (slab >= 0) {
        const uint8_t* src = a.k_pool + ((size_t)slab * kMqPage + ct % kMqPage) * (D / 2);
#pragma unroll
        for (int q = 0; q < D / 32; ++q)
          cp_async16(codes_of(i) + ct * kRow + ((q ^ code_swizzle<D>(ct)) << 4), src + 16 * q);
      }
      float* sz = scales_of(i);
#pragma unroll 1
      for (uint32_t left = d.slots; left; left &= left - 1) {
        const int slot = __ffs(left) - 1;
        const float* src = a.sz_pool + (size_t)d.home[slot] * (2 * D);
#pragma unroll
        for (int ch = 0; ch < D; ch += 128) {
          if (D >= 128 || ct < D) {
            cp_async4(sz + slot * (2 * D) + ch + ct, src + ch + ct);
            cp_async4(sz + slot * (2 * D) + D + ch + ct, src + D + ch + ct);
          }
        }
      }
      cp_async_commit();
    };
    bool ok = true;
    // (the first turn, before the group's first tile, only starts that tile's copies)
#pragma unroll 1
    for (int i = grp - 2; i < n_tiles; i += 2) {
      const int ds = i & (kDesc - 1), next = i + 2;
      const TileDesc& d = sh.desc[ds];
      const int flags = i >= 0 ? d.flags : 0;
      const bool draft = flags & kDraftTile;
      float* scales = scales_of(i);
      bool scaled = false;
      if (i >= 0) {
        // Scale and zero point, in place: a code c enters as 1 + c / 128 (its bits in
        // the mantissa), so a key is (1 + c / 128) e + z with e = 128 s, z = -zp s - e.
        bool odd = false;  // a group outside float16's range
        cp_async_wait<0>();
#pragma unroll 1
        for (uint32_t left = ok ? d.slots : 0u; left; left &= left - 1) {
          float* sz = scales + (__ffs(left) - 1) * (2 * D) + ct;
          float key_top = 0.f;
#pragma unroll
          for (int ch = 0; ch < D; ch += 128) {
            if (D >= 128 || ct < D) {
              const float s = sz[ch], z = -sz[D + ch] * s;
              key_top = fmaxf(key_top, fmaxf(finite_abs(z), finite_abs(fmaf(15.f, s, z))));
              sz[ch] = 128.f * s;
              sz[D + ch] = fmaf(-128.f, s, z);
            }
          }
          // (a warp judges its own channels: too small there alone costs time, no more)
          odd |= key_top >= kHalfRoom || ((D >= 128 || ct < D) && !__any_sync(0xffffffffu, key_top >= kHalfLow));
        }
        // The keys of tile i - 2 have been multiplied. A new stream's queries replace
        // the last one's: every product with those is done. (In this order: a wait
        // tells a phase from its neighbours only, and tile i - 3's has to be over
        // before tile i - 1's is asked for.)
        ok = ok && tc_wait(&sh.kh_empty[i & 1], (i / 2 + 1) & 1, a.status);
        if (ok && (flags & kFirst) && i > 0) ok = tc_wait(&sh.kh_empty[(i - 1) & 1], ((i - 1) / 2) & 1, a.status);
        // Keys outside float16's range take a power of two per group.
        if (named_bar_or(bar, 128, !ok || odd)) {
          // (uniform over the group: its warps meet in named barriers)
          if (named_bar_or(bar, 128, !ok)) break;
          scaled = true;
        }
        tc_fence_after();
      }
      if (T::NB > 1 && next < n_tiles) {
        ok = __all_sync(0xffffffffu, tc_wait(&sh.desc_full[next % kDesc], (next / kDesc) & 1, a.status));
        if (ok) prefetch(sh.desc[next % kDesc], next);
      }
      if (i < 0) {
        if (T::NB > 1) continue;
        if (next < n_tiles) {
          ok = __all_sync(0xffffffffu, tc_wait(&sh.desc_full[next % kDesc], (next / kDesc) & 1, a.status));
          if (ok) prefetch(sh.desc[next % kDesc], next);
        }
        continue;
      }
      if (flags & kFirst) load_queries<D, NR, VK>(a, ds, ct);
      const uint32_t keys = tm + lanes + T::COLS_K + (i & 1) * (D / 2);
      if (draft) {
        scaled = draft_keys<D, NR, VK>(a, ds, keys, ct, bar);
      } else {
        const char* codes = codes_of(i);
        if (scaled) convert_scaled<D, NR>(ds, codes, scales, keys, ct);
        else convert_keys<D, false>(d, codes, scales, keys, ct, 1.f, 1.f);
      }
      if (ct == 0) sh.scaled[ds] = scaled;
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.kh_full[i & 1]);
        mbar_arrive(&sh.desc_empty[ds]);
      }
      if (T::NB == 1) {
        named_bar_sync(bar, 128);
        if (next < n_tiles) {
          ok = __all_sync(0xffffffffu, tc_wait(&sh.desc_full[next % kDesc], (next / kDesc) & 1, a.status));
          if (ok) prefetch(sh.desc[next % kDesc], next);
        }
      }
    }
    cp_async_wait<0>();
  } else {
    // ------------------------------------------------------------ softmax
    // Logits are read as fragments: thread (g, t) of a warp holds tokens g, g + 8 of
    // the warp's two pages and rows 8 i + 2 t, + 1, so a thread's rows are few: their
    // references and sums stay in its registers (as broadcasts from shared memory they
    // would cost a cycle per row and warp, as many as the exponentials do).
    constexpr int NC = T::NC, NI = NC / 8;     // rows of the warpgroup; pairs of rows of a thread
    constexpr int LI = NI < 4 ? NI : 4;        // pairs per load
    const int wg = warp / 4, quarter = warp % 4, tok = quarter * 32 + lane, c0 = wg * NC;
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int bar = kBarGroup + wg;
    float nref[NI][2], l[NI][2];               // minus the references; sums
    bool failed = false, started = false;      // a wait ran out; O^T of the segment holds something
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      nref[j][0] = nref[j][1] = -kNoRef;
      l[j][0] = l[j][1] = 0.f;
    }
#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
      const int ds = i % kDesc, sb = i & 1, pb = i % T::NP;
      // Every thread waits. A timeout is made uniform over the warpgroup with the
      // tile's vote alone: until then the tile goes on with what it has, so no barrier
      // of the warpgroup (they share none) ever waits for a warp that has left.
      const bool ok = tc_wait(&sh.desc_full[ds], (i / kDesc) & 1, a.status);
      failed |= !ok;
      const TileDesc& d = sh.desc[ds];
      const int flags = ok ? d.flags : 0, sg = ok ? d.seg : 0;
      const bool masked = flags & kMasked;
      failed |= !tc_wait(&sh.s_full[sb], (i / 2) & 1, a.status);
      tc_fence_after();
      if (flags & kFirst) {
        started = false;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          nref[j][0] = nref[j][1] = -kNoRef;
          l[j][0] = l[j][1] = 0.f;
        }
      }
      const uint32_t s_addr = tm + lanes + sb * NR + c0;
      if (sh.scaled[ds] | sh.qscaled[sg]) scale_tile<D, NR>(ds, s_addr, c0, tok);
      if (masked) mask_tile<D, NR>(a, ds, s_addr, c0, tok);
      // pass 1: does some logit exceed its row's reference by more than kLazy? (Up to
      // 32 rows' logits stay in registers for pass 2.)
      constexpr bool kHeld = LI == NI;
      uint32_t x[2][4 * LI];
      float over = -INFINITY;
#pragma unroll
      for (int j0 = 0; j0 < NI; j0 += LI) {
        tc_ld_frag(x[0], x[1], s_addr + 8 * j0);
#pragma unroll
        for (int j = 0; j < LI; ++j) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t* xx = &x[q / 2][4 * j + 2 * (q % 2)];
            float y0, y1;
            fma2(y0, y1, __uint_as_float(xx[0]), __uint_as_float(xx[1]), kLog2e, kLog2e, nref[j0 + j][0], nref[j0 + j][1]);
            over = fmax3f(over, y0, y1);
          }
        }
      }
      const bool raised = named_bar_or(bar, 128, over > kLazy || failed);  // (the warpgroup's answer)
      if (raised) {
        if (named_bar_or(bar, 128, failed)) break;
        RowState<NI> rows;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            rows.nref[j][e] = nref[j][e];
            rows.l[j][e] = l[j][e];
          }
        }
        rows = raise_references<D, NR>(a, rows, s_addr, tm + lanes + T::COLS_O + c0, c0,
                                       quarter, lane, started ? (i - 1) % T::NP : -1, ((i - 1) / T::NP) & 1, bar);
        failed |= rows.failed;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            nref[j][e] = rows.nref[j][e];
            l[j][e] = rows.l[j][e];
          }
        }
      }
      // pass 2: weights
      failed |= !tc_wait(&sh.p_empty[pb], (i / T::NP + 1) & 1, a.status);
      char* prow = smem + T::P_OFF + pb * T::P + (quarter * 32 + g) * 128 + 4 * t4;
#pragma unroll
      for (int j0 = 0; j0 < NI; j0 += LI) {
        if (!kHeld) tc_ld_frag(x[0], x[1], s_addr + 8 * j0);
#pragma unroll
        for (int j = 0; j < LI; ++j) {
          const int col = c0 + 8 * (j0 + j);
          char* at = prow + (col / 64) * (kTile * 128) + (((col / 8) % 8 ^ g) << 4);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t* xx = &x[q / 2][4 * j + 2 * (q % 2)];
            float y0, y1;
            fma2(y0, y1, __uint_as_float(xx[0]), __uint_as_float(xx[1]), kLog2e, kLog2e, nref[j0 + j][0], nref[j0 + j][1]);
            y0 = exp2_fast(y0);
            y1 = exp2_fast(y1);
            const uint32_t w2 = pack_weights<VK>(y0, y1);
            *reinterpret_cast<uint32_t*>(at + q * 8 * 128) = w2;
            // (the sums take what the product takes: a row's weights sum to one)
            widen2<VK>(w2, y0, y1);
            add2_rn(l[j0 + j][0], l[j0 + j][1], l[j0 + j][0], l[j0 + j][1], y0, y1);
          }
        }
      }
      if (masked && wg == 0) failed |= !clear_values<D, NR, VK>(a, ds, i, tok);
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      const bool last = flags & kLast;
      if (lane == 0) {
        mbar_arrive(&sh.s_empty[sb]);
        mbar_arrive(&sh.p_full[pb]);
        if (!last) mbar_arrive(&sh.desc_empty[ds]);
      }
      started = true;
      if (last) {
        // ---- epilogue: O^T, a lane a channel, over the sums of the weights ----
        if (raised) named_bar_sync(bar, 128);  // (every warp has read the maxima where the sums go)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = l[j][e];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const int r = c0 + 8 * j + 2 * t4 + e;
            if (g == 0) {
              sh.part[quarter][r] = x;
              if (quarter == 0) sh.ref[r] = -nref[j][e];
            }
          }
        }
        // (the product waited for every warp's weights: the list of odd values is complete)
        failed |= !tc_wait(&sh.p_empty[pb], (i / T::NP) & 1, a.status);
        named_bar_sync(bar, 128);
        finish_stream<D, NR, VK>(a, ds, tm + lanes, c0, tok, bar);
        if (lane == 0) mbar_arrive(&sh.desc_empty[ds]);
      }
    }
  }
  // all roles meet; tensor memory is freed on every path
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(T::COLS));
  }
}

cudaError_t encoder(PFN_cuTensorMapEncodeTiled_v12000* fn) {
  static std::mutex mu;
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  std::lock_guard<std::mutex> lk(mu);
  if (!encode) {
    cudaDriverEntryPointQueryResult qr;
    void* p = nullptr;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr);
    if (e != cudaSuccess) return e;
    if (qr != cudaDriverEntryPointSuccess || !p) return cudaErrorNotSupported;
    encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  *fn = encode;
  return cudaSuccess;
}

// [outer][rows][chunks of 64 channels] 16-bit values as boxes of one outer
// entry, 16 rows and every chunk, 128-byte swizzled.
cudaError_t value_map(CUtensorMap* map, const void* base, int vk, int dim, uint64_t rows, uint64_t row_bytes,
                      uint64_t outer, uint64_t outer_bytes) {
  PFN_cuTensorMapEncodeTiled_v12000 encode;
  const cudaError_t e = encoder(&encode);
  if (e != cudaSuccess) return e;
  const cuuint64_t dims[4] = {64, rows, (cuuint64_t)dim / 64, outer};
  const cuuint64_t strides[3] = {row_bytes, 128, outer_bytes};
  const cuuint32_t box[4] = {64, kMqPage, (cuuint32_t)dim / 64, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, vk == INT4KV_VALUES_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                            4, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int D, int NR, int VK>
cudaError_t launch(const MultiQueryArgs& args, int sms, void* ws, size_t ws_bytes, cudaStream_t stream) {
  using T = Tc<D, NR>;
  constexpr size_t kBytes = T::END + sizeof(TcShared<NR>);
  static_assert(T::END + sizeof(TcShared<NR>) <= 227 * 1024, "shared memory");
  constexpr auto kern = multi_query_tc_kernel<D, NR, VK>;
  int per_sm = 0;
  cudaError_t e = mq_occupancy<kern>(T::THREADS, kBytes, &per_sm);
  if (e != cudaSuccess) return e;
  MultiQueryArgs a = args;
  if (!mq_workspace(a, ws, ws_bytes, sms, Record<NR, D>::kFloats)) return cudaErrorInvalidValue;
  CUtensorMap vmap, dmap;
  const uint64_t row = (uint64_t)D * 2;
  if ((long long)a.num_pages * a.kv_heads > 0x7fffffffll) return cudaErrorInvalidValue;  // a TMA coordinate
  e = value_map(&vmap, a.v_pool, VK, D, kMqPage, row, (uint64_t)a.num_pages * a.kv_heads, kMqPage * row);
  if (e != cudaSuccess) return e;
  if (a.vd) e = value_map(&dmap, a.vd, VK, D, a.total_rows, row * a.kv_heads, a.kv_heads, row);
  else dmap = vmap;
  if (e != cudaSuccess) return e;
  e = mq_launch_pdl(kern, dim3(sms), dim3(T::THREADS), kBytes, stream, a, vmap, dmap);
  if (e != cudaSuccess) return e;
  return mq_launch_pdl(merge_records_kernel<NR, D>, dim3(sms - 1, (NR + kMergeWarps - 1) / kMergeWarps),
                       dim3(kMergeWarps * 32), 0, stream, a);
}

// Rows of one kv head's chunk: the smallest of 16, 32, 64, 128 that holds them
// (head_dim 256: at most 64, the most its shared memory holds). More than 64 rows go in
// chunks of 64 all the same where chunks of 128 would be `few` streams: fewer than half of
// the CTAs, and with little to do for each (units of 128-row tiles a CTA, at most). A tile
// of 64 rows is not half as dear, but a stream's start and end are, and where a stream is
// shared by many CTAs each of them pays for those. (64 against 128 rows a chunk, bfloat16,
// head_dim 128, 8 kv heads: 64 streams, 128 rows: 8 x 300 31 and 43 us, 8 x 4096 71 and
// 75, 8 x 6000, 22 units a CTA, 89 and 91, but 8 x 8192, 30 units, 110 and 103. 32 streams of
// 256 rows: 2 x 2048 38 and 43. 128 streams of 256 rows: 8 x 300 51 and 48, 8 x 1000 73 and
// 67, 8 x 4096 124 and 111. 192 streams and more: 24 x 1000 105 and 87, 32 x 8192 378 and 301.)
constexpr double kFewUnits = 24;
int rows_of(long long rows, int dim, bool few) {
  if (rows <= 16) return 16;
  if (rows <= 32) return 32;
  return rows <= 64 || dim == 256 || few ? 64 : 128;
}
// From the sizes that the host knows: the table's width, or the window, for every sequence.
bool few_streams(const MultiQueryArgs& a, long long rows, int sms) {
  double pages = a.max_pages;
  if (a.window > 0) pages = std::min(pages, ((double)a.window + a.sinks) / kMqPage + 2);
  const double streams = (double)a.batch * a.kv_heads * (double)((rows + 127) / 128);
  return 2 * streams < sms && streams * (std::ceil(pages / kTilePages) + 1 + kStreamUnits + kDraftUnits) / sms < kFewUnits;
}

template <int D, int NR>
cudaError_t launch_kind(const MultiQueryArgs& a, int sms, void* ws, size_t n, cudaStream_t st) {
  return a.qk == INT4KV_VALUES_F16 ? launch<D, NR, INT4KV_VALUES_F16>(a, sms, ws, n, st)
                                   : launch<D, NR, INT4KV_VALUES_BF16>(a, sms, ws, n, st);
}

template <int D>
cudaError_t launch_rows(int nr, const MultiQueryArgs& a, int sms, void* ws, size_t n, cudaStream_t st) {
  if (nr == 16) return launch_kind<D, 16>(a, sms, ws, n, st);
  if (nr == 32) return launch_kind<D, 32>(a, sms, ws, n, st);
  if constexpr (D < 256) {
    if (nr == 128) return launch_kind<D, 128>(a, sms, ws, n, st);
  }
  return launch_kind<D, 64>(a, sms, ws, n, st);
}

}  // namespace

namespace i4kv {

double multi_query_tc_units(const MultiQueryArgs& a, int dim) {
  const long long rows = (long long)std::max(1, a.max_drafts) * a.group_q;
  // (with the larger choice of rows: the smaller is for a few units a CTA)
  return mq_most_units(a, rows, rows_of(rows, dim, false), kTilePages, kStreamUnits + kDraftUnits);
}

size_t multi_query_tc_workspace(int dim, long long rows, int sms) {
  const int nr = rows_of(rows, dim, false);  // (the larger choice)
  return mq_workspace_bytes(sms, 2 * nr + nr * dim);
}

cudaError_t multi_query_tc(const MultiQueryArgs& a, int dim, int sms, void* ws, size_t ws_bytes, cudaStream_t stream) {
  const long long rows = (long long)std::max(1, a.max_drafts) * a.group_q;
  const int nr = rows_of(rows, dim, few_streams(a, rows, sms));
  if (dim == 64) return launch_rows<64>(nr, a, sms, ws, ws_bytes, stream);
  if (dim == 128) return launch_rows<128>(nr, a, sms, ws, ws_bytes, stream);
  return launch_rows<256>(nr, a, sms, ws, ws_bytes, stream);
}

}  // namespace i4kv
