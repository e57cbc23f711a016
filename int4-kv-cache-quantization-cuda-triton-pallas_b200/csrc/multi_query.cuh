// Work decomposition shared by the kernels in which several queries of a
// sequence attend over its paged INT4 cache (drafted trees, sliding windows).
//
// Sequence b has `rows` query rows per kv head, row = draft * G + (query head
// of the group), in chunks of NR rows; a stream is one (b, kv head, chunk). Its
// work is a list of tiles: the blocks of TP pages (from multiples of TP, so that a
// block lies in one quantization group wherever groups are that long) that hold
// visible pages, those of the sinks and those of the window, then the drafted
// tokens. The streams' tiles are laid end to end and
// every CTA takes one contiguous run of equal cost, whatever the lengths are: a
// tile costs one unit, and what a stream costs besides (its queries, its end, and
// drafts' masks) is counted as a few units before its first tile. A stream inside one
// run is finished by its CTA; of a shared stream each CTA leaves a record (m, l, acc)
// per row, and the first of them a note of who shares it (RunTail), by which
// merge_records_kernel, one block per run, combines them. Records and notes need
// no counters, so the workspace carries nothing between launches, and their order
// of combination is fixed: equal inputs give equal bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "run_tail.h"
#include "../../include/int4kv_b200.h"

namespace i4kv {

constexpr int kMqPage = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMqMaxDrafts = INT4KV_MAX_DRAFTS;

struct MultiQueryArgs {
  const void* q;               // [rows, Hq, D] of kind qk
  const void* kd;              // [rows, Hkv, D] drafted keys / values of kind qk (tree only)
  const void* vd;
  const int64_t* mask;         // [rows] bit u: draft u of the same sequence is visible (tree only)
  const int32_t* offs;         // [B+1] rows of each sequence (null: one row each, already cached)
  const uint8_t* k_pool;
  const void* v_pool;
  const float* sz_pool;
  const int32_t* block_table;
  const int32_t* seq_lens;
  void* out;                   // [rows, Hq, D] of kind qk
  RunTail* tails;              // one per CTA
  float* recs;                 // two records per CTA
  uint32_t* status;
  int qk, batch, kv_heads, group_q, total_rows, max_drafts;
  int max_pages, num_pages, group_pages;
  int window, sinks;           // window 0: the whole cache
};

// What one sequence asks for.
struct SeqWork {
  int len, drafts, row0, rows, chunks;
  int pos0;                    // position of a query without drafted ancestors
  int pages, sink_pages, win_page;  // visible pages: [0, sink_pages) and [win_page, pages)
  int sink_blocks, win_block;       // and the blocks that hold them: [0, sink_blocks), [win_block, ..)
  int cache_tiles, tiles;
};

I4KV_DEVINL void mq_status(uint32_t* status, uint32_t bits) {
  if (status) atomicOr(status, bits);
}

// (Not inlined: it runs once per sequence, and every kernel calls it from
// several places.)
template <int NR, int TP>
__device__ __noinline__ SeqWork seq_work(const MultiQueryArgs& a, int b, bool report) {
  SeqWork w;
  const int cap = a.max_pages * kMqPage;  // < 2^31 - 128 (checked on the host)
  int len = a.seq_lens[b];
  bool bad = len < 0 || len > cap;
  w.len = len < 0 ? 0 : (len > cap ? cap : len);
  if (a.offs) {
    const int lo = a.offs[b], hi = a.offs[b + 1];
    const long long n = (long long)hi - lo;
    const bool ok = lo >= 0 && n >= 0 && n <= a.max_drafts && hi <= a.total_rows;
    bad |= !ok;
    w.row0 = ok ? lo : 0;
    w.drafts = ok ? (int)n : 0;
    w.rows = w.drafts * a.group_q;
    w.pos0 = w.len;
  } else {
    w.row0 = b;
    w.drafts = 0;
    w.rows = a.group_q;
    w.pos0 = w.len - 1;
  }
  if (bad && report) mq_status(a.status, kStatusBadLength);
  w.chunks = (w.rows + NR - 1) / NR;
  w.pages = (w.len + kMqPage - 1) / kMqPage;
  w.sink_pages = 0;
  w.win_page = 0;
  if (a.window > 0) {
    const int lo = w.pos0 - a.window + 1;  // first windowed position of the lowest query
    if (lo > 0) {
      w.win_page = min(lo / kMqPage, w.pages);
      w.sink_pages = (int)(((long long)min(a.sinks, w.len) + kMqPage - 1) / kMqPage);
    }
  }
  w.sink_blocks = (w.sink_pages + TP - 1) / TP;
  w.win_block = w.win_page / TP;
  const int blocks = (w.pages + TP - 1) / TP;
  if (w.win_page >= w.pages) w.win_block = blocks;  // nothing in the window
  if (w.sink_blocks >= w.win_block) {                // one run of blocks
    w.sink_blocks = 0;
    if (w.sink_pages > 0) w.win_block = 0;
  }
  w.cache_tiles = w.sink_blocks + blocks - w.win_block;
  w.tiles = w.rows > 0 ? w.cache_tiles + (w.drafts + TP * kMqPage - 1) / (TP * kMqPage) : 0;
  return w;
}

// Page j of cache tile i, and whether some query sees it.
template <int TP>
I4KV_DEVINL int tile_page(const SeqWork& w, int i, int j) {
  return (i < w.sink_blocks ? i : i - w.sink_blocks + w.win_block) * TP + j;
}
I4KV_DEVINL bool page_visible(const SeqWork& w, int pg) {
  return pg < w.pages && (pg < w.sink_pages || pg >= w.win_page);
}

// Place of one tile in the end-to-end order.
struct TileAt {
  int b, head, chunk, tile;
};

// Unit at which run c of n begins, and the run of a unit. (Counts of units fit 31
// bits: checked on the host for the largest lengths.)
I4KV_DEVINL int run_start(int c, int total, int n) { return (int)((long long)c * total / n); }
I4KV_DEVINL int run_of(int u, int total, int n) { return (int)((((long long)u + 1) * n - 1) / total); }

static __device__ __noinline__ TileAt tile_at(const MultiQueryArgs& a, const SeqWork w, int b, int rem) {
  TileAt p;
  const int per_head = w.tiles * w.chunks;
  p.b = b;
  p.head = rem / per_head;
  const int r = rem - p.head * per_head;
  p.chunk = r / w.tiles;
  p.tile = r - p.chunk * w.tiles;
  return p;
}

// A CTA's run: `tiles` tiles, the first of them tile `rem` of sequence b; all runs
// together have `total` units, and this one's end before unit `end`.
struct RunPlan {
  int total, runs, end, tiles, b, rem;
};

// ... by one converged warp, from the lengths alone (every CTA finds its own). A
// stream costs EXTRA units besides its tiles, DRAFT more with drafts.
template <int NR, int TP, int EXTRA, int DRAFT>
__device__ __noinline__ RunPlan plan_run(const MultiQueryArgs& a, int cta, int ctas) {
  const int lane = threadIdx.x & 31;
  RunPlan p = {};
  // units and tiles of this lane's sequence of the 32 from `base` on
  int tiles = 0, units = 0, extra = 0, streams = 0;
  auto of_sequence = [&](int base, bool report) {
    tiles = units = streams = extra = 0;
    if (base + lane < a.batch) {
      const SeqWork w = seq_work<NR, TP>(a, base + lane, report);
      if (w.tiles > 0) {
        tiles = w.tiles;
        extra = EXTRA + (w.drafts > 0 ? DRAFT : 0);
        streams = w.chunks * a.kv_heads;
        units = streams * (tiles + extra);
      }
    }
  };
#pragma unroll 1
  for (int base = 0; base < a.batch; base += 32) {
    of_sequence(base, cta == 0);
    p.total += __reduce_add_sync(0xffffffffu, units);
  }
  p.runs = min(ctas, p.total);
  if (cta >= p.runs) return p;
  const int begin = run_start(cta, p.total, p.runs);
  p.end = run_start(cta + 1, p.total, p.runs);
  // tiles before the run's first unit and before its end
  int before = 0, tiles_before = 0, first_tile = 0, last_tile = -1;
#pragma unroll 1
  for (int base = 0; base < a.batch && last_tile < 0; base += 32) {
    if (a.batch > 32) of_sequence(base, false);
    int iu = units, it = streams * tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, iu, o), t = __shfl_up_sync(0xffffffffu, it, o);
      if (lane >= o) {
        iu += u;
        it += t;
      }
    }
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const int u = k ? p.end : begin;
      // the sequence of unit u; for the run's end, of the unit before it
      const uint32_t hit = __ballot_sync(0xffffffffu, before + iu > (k ? u - 1 : u) && before + iu - units <= (k ? u - 1 : u));
      if (!hit) continue;
      const int l = __ffs(hit) - 1, off = u - before - (iu - units), per = tiles + extra;
      // (lane l's own numbers) whole streams before u, then tiles of the one u lies in
      const int whole = per > 0 ? off / per : 0;
      const int in_seq = whole * tiles + max(0, off - whole * per - extra);
      const int at = __shfl_sync(0xffffffffu, in_seq, l);
      const int all = tiles_before + __shfl_sync(0xffffffffu, it - streams * tiles, l) + at;
      if (k) {
        last_tile = all;
      } else {
        first_tile = all;
        p.b = base + l;
        p.rem = at;
      }
    }
    before += __shfl_sync(0xffffffffu, iu, 31);
    tiles_before += __shfl_sync(0xffffffffu, it, 31);
  }
  p.tiles = last_tile - first_tile;
  return p;
}

// The note of a run's last stream (tile `t` of it is the run's last).
static __device__ __noinline__ void note_tail(const MultiQueryArgs& a, int cta, const RunPlan p, const SeqWork w, const TileAt t,
                                              int nr) {
  RunTail n = {};
  const int first = p.tiles - 1 - t.tile;  // the stream's first tile, of the run's
  if (t.tile + 1 < w.tiles && first >= 0) {
    n.rows = w.rows;
    n.row0 = w.row0;
    n.head = t.head;
    n.first_row = t.chunk * nr;
    n.slot = 2 * cta + (first > 0 ? 1 : 0);
    n.last = run_of(p.end + w.tiles - 2 - t.tile, p.total, p.runs);  // (the units from here on are its tiles)
  }
  a.tails[cta] = n;
}

// Step to the next stream; `w` follows the sequence. False past the last one.
template <int NR, int TP>
I4KV_DEVINL bool next_stream(const MultiQueryArgs& a, SeqWork& w, TileAt& p) {
  p.tile = 0;
  if (++p.chunk < w.chunks) return true;
  p.chunk = 0;
  if (++p.head < a.kv_heads) return true;
  p.head = 0;
  while (++p.b < a.batch) {
    w = seq_work<NR, TP>(a, p.b, false);
    if (w.tiles > 0 && w.rows > 0) return true;
  }
  return false;
}

// Element offset of row r of a stream's chunk in q / out.
I4KV_DEVINL size_t row_offset(const MultiQueryArgs& a, const SeqWork& w, int head, int rr, int D) {
  const int t = rr / a.group_q, g = rr - t * a.group_q;
  return ((size_t)(w.row0 + t) * a.kv_heads * a.group_q + (size_t)head * a.group_q + g) * D;
}

// Drafted ancestors of draft t (its position behind the cache).
I4KV_DEVINL int draft_depth(uint64_t word, int t, int drafts) {
  const uint64_t real = drafts >= 64 ? ~0ull : (1ull << drafts) - 1;
  return __popcll(word & real & ~(1ull << t));
}

template <int N>
I4KV_DEVINL void load_f32(const void* base, int kind, size_t i, float (&x)[N]) {
  if (kind == INT4KV_VALUES_F32) {
    const float* p = static_cast<const float*>(base) + i;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 v = *reinterpret_cast<const float2*>(p + j);
      x[j] = v.x;
      x[j + 1] = v.y;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + i;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p + j);
      if (kind == INT4KV_VALUES_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        x[j] = f.x;
        x[j + 1] = f.y;
      } else {
        x[j] = __uint_as_float(w << 16);
        x[j + 1] = __uint_as_float(w & 0xFFFF0000u);
      }
    }
  }
}

I4KV_DEVINL void store2(void* base, int kind, size_t i, float x, float y) {
  if (kind == INT4KV_VALUES_F32) {
    *reinterpret_cast<float2*>(static_cast<float*>(base) + i) = make_float2(x, y);
  } else if (kind == INT4KV_VALUES_F16) {
    *reinterpret_cast<__half2*>(static_cast<__half*>(base) + i) = __floats2half2_rn(x, y);
  } else {
    *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(base) + i) = __floats2bfloat162_rn(x, y);
  }
}

// A CTA's record of one stream: m [NR] (natural units), l [NR], acc [NR, D].
template <int NR, int D>
struct Record {
  static constexpr int kFloats = 2 * NR + NR * D;
};

// Rows of sequences that see nothing (a window over an empty cache) are zeros.
template <int NR, int TP, int D>
__device__ __noinline__ void zero_idle_rows(const MultiQueryArgs& a) {
#pragma unroll 1
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    const SeqWork w = seq_work<NR, TP>(a, b, false);
    if (w.tiles > 0 || w.rows == 0) continue;
    const int n = a.kv_heads * a.group_q * D;  // one row a sequence
#pragma unroll 1
    for (int i = 2 * threadIdx.x; i < n; i += 2 * blockDim.x)
      store2(a.out, a.qk, (size_t)w.row0 * n + i, 0.f, 0.f);
  }
}

I4KV_DEVINL void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

I4KV_DEVINL float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Units of all streams together at most, in chunks of `nr` rows and tiles of `tp` pages;
// the kernels count them in 31 bits. (From the table's width, or the window and the
// sinks, for every sequence: what the host knows.)
inline double mq_most_units(const MultiQueryArgs& a, long long rows, int nr, int tp, int extra) {
  const auto blocks = [&](long long pages) { return (double)((pages + tp - 1) / tp); };
  double tiles = blocks(a.max_pages);
  if (a.window > 0)  // (their first and last pages, and blocks, may be parts)
    tiles = std::min(tiles, blocks(a.window / kMqPage + 2) + 1 + blocks(a.sinks / kMqPage + 1));
  tiles += blocks((a.max_drafts + kMqPage - 1) / kMqPage) + extra;
  return tiles * (double)((rows + nr - 1) / nr) * a.batch * a.kv_heads;
}
constexpr double kMqMostUnits = 2147483647.;

// Workspace of `runs` runs: their notes, then two records each.
inline size_t mq_workspace_bytes(int runs, int record_floats) {
  return (size_t)runs * sizeof(RunTail) + (size_t)runs * 2 * record_floats * 4;
}
inline bool mq_workspace(MultiQueryArgs& a, void* ws, size_t bytes, int runs, int record_floats) {
  if (bytes < mq_workspace_bytes(runs, record_floats)) return false;
  a.tails = static_cast<RunTail*>(ws);
  a.recs = reinterpret_cast<float*>(a.tails + runs);
  return true;
}

constexpr int kMergeWarps = 8;

// Combine the records of the streams that lie across runs: block x the one that run
// x began and did not end (if any), blocks y kMergeWarps rows each, one warp a row.
// Plain float32 with weights e^(m_i - M): a handful of terms.
template <int NR, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_records_kernel(MultiQueryArgs a) {
  grid_dependency_wait();
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const int4 n0 = __ldcg(reinterpret_cast<const int4*>(a.tails + c));
  const int2 n1 = __ldcg(reinterpret_cast<const int2*>(a.tails + c) + 2);
  const RunTail n = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, {}};
  // (one block less than runs)
  if (!tail_in_range(n, c, gridDim.x + 1, a.total_rows, a.kv_heads, a.group_q)) return;
  const int row0 = n.row0, head = n.head, slot = n.slot, last = n.last;
  const int r = blockIdx.y * kMergeWarps + (threadIdx.x >> 5), rr = n.first_row + r;
  if (rr >= n.rows) return;
  constexpr int kRec = Record<NR, D>::kFloats;
  auto record = [&](int i) { return a.recs + (size_t)(i == c ? slot : 2 * i) * kRec; };
  float M = -INFINITY;
#pragma unroll 1
  for (int i = c + lane; i <= last; i += 32) M = fmaxf(M, __ldcg(record(i) + r));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float L = 0.f, o[D / 32];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) o[k] = 0.f;
  if (M != -INFINITY) {
#pragma unroll 2
    for (int i = c; i <= last; ++i) {
      const float* rec = record(i);
      const float e = exp2_fast((__ldcg(rec + r) - M) * kLog2e);
      L = fmaf(__ldcg(rec + NR + r), e, L);
      const float* acc = rec + 2 * NR + (size_t)r * D;
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(acc + 64 * k + 2 * lane));
        o[2 * k] = fmaf(x.x, e, o[2 * k]);
        o[2 * k + 1] = fmaf(x.y, e, o[2 * k + 1]);
      }
    }
  }
  const float inv = 1.f / fmaxf(L, 1e-10f);
  const int t = rr / a.group_q;
  const size_t to = (((size_t)(row0 + t) * a.kv_heads + head) * a.group_q + (rr - t * a.group_q)) * D;
#pragma unroll
  for (int k = 0; k < D / 64; ++k) store2(a.out, a.qk, to + 64 * k + 2 * lane, o[2 * k] * inv, o[2 * k + 1] * inv);
}

// Resident CTAs per SM of kernel Kern with `smem` dynamic bytes, once per kernel and
// device (also raises the kernel's shared-memory limit there).
template <auto Kern>
cudaError_t mq_occupancy(int threads, size_t smem, int* per_sm) {
  static std::mutex mu;
  static int known[64];  // 0: not asked yet
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lk(mu);
  if (!known[dev]) {
    e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    int n = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kern, threads, smem);
    if (e != cudaSuccess) return e;
    if (n < 1) return cudaErrorInvalidConfiguration;
    known[dev] = n;
  }
  *per_sm = known[dev];
  return cudaSuccess;
}

// Launch with programmatic stream serialization: the kernel's CTAs may be
// placed while its predecessor ends; it waits for it before it reads.
template <typename... KArgs, typename... Args>
cudaError_t mq_launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                          Args... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace i4kv
