// Several queries of a sequence over its paged INT4 cache in float32: drafted
// trees (int4kv_paged_tree_decode) and sliding windows with sinks
// (int4kv_paged_window_decode).
//
// Math: per row, logits x_j = sum_c q_c (code_jc s_c - zp_c s_c) over the
// visible cached tokens and q . k over the visible drafts, one pass with the
// running maximum m and sum l, out = sum_j 2^((x_j - m) log2 e) v_j / l. Keys
// are dequantized in registers, once for the NR rows of a CTA; products and
// sums are float32 in paired instructions (two lanes of work per issue). Each of
// eight warps sums its share of the tokens, where registers allow a tile's values
// from zero first, so a long cache costs several short sums instead of one long
// one: the error stays near 2^-24 sqrt(tokens / 64), not 2^-24 sqrt(tokens).
//
// A tile is 64 tokens. A warp takes 8 of them from the logits to the values by
// itself, with its own running maxima, sums and outputs, and the eight warps meet
// only when the stream ends: nothing in a tile waits for another warp but the
// copies do (a ninth warp issues them, two stages, as soon as all have left one).
//   logits: 8 lanes share a token, a lane holds two tokens and 8 of every 64
//     channels, so a scale or query read from shared memory serves both (the upper
//     four lanes take their second four channels first: the eight 16-byte reads of
//     a token's lanes then hit different banks); a reduce-scatter leaves each lane one
//     token's logits of NR / 4 rows.
//   values: a lane holds D / 32 channels of all NR rows; the weights come as
//     broadcasts from shared memory.
// Which of bytes and arithmetic bounds it depends on NR: a tile costs NR * 2 * D *
// 64 fused multiply-adds whatever the rows' count, so NR is the smallest of 1, 4, 8,
// 16 that holds the rows of one kv head (head_dim 256: at most 8, what its
// accumulators leave of the registers).
// Measured (B200, 32 heads, head_dim 128, float32 values): window of 2000 over 32 x
// 4096 tokens 217 to 234 us on different machines (5.1 to 5.5 TB/s, HBM and the logits'
// arithmetic); 4 drafts over 8 x 2048 90 us (3.4 TB/s, issue and shared-memory reads).
// With bfloat16 values, half the bytes, 221 and 92 us: the arithmetic alone. 16 drafts of
// 32 query heads over 8, 8 x 2048: 257 us, four chunks of 16 rows that each read and
// dequantize the cache again.
#include <algorithm>

#include "multi_query.cuh"

using namespace i4kv;

namespace {

constexpr int kWarps = 8, kConsumers = 32 * kWarps, kThreads = kConsumers + 32;
constexpr int kStreamUnits = 1, kDraftUnits = 1;  // what a stream costs besides its tiles, in tiles
constexpr int kMaxPerSm = 4;                  // CTAs per SM the workspace is sized for
constexpr uint64_t kWaitNs = 2000000000ull;  // bounded waits: 2 s

template <int D, int NR, int VK>
struct Shape {
  static constexpr int TOK = 64, TP = TOK / kMqPage;
  static constexpr int VB = VK == INT4KV_VALUES_F32 ? 4 : 2;
  static constexpr int V_BYTES = TOK * D * VB, K_BYTES = TOK * D / 2, SZ_BYTES = TP * 2 * D * 4;
  static constexpr int STAGE = V_BYTES + K_BYTES + SZ_BYTES;
  static constexpr int KB = NR <= 4 ? kWarps : 1;  // copies of the outputs the warps' sums meet in
  static constexpr int Q_OFF = 2 * STAGE;
  static constexpr int O_OFF = Q_OFF + NR * D * 4;
  static constexpr int P_OFF = O_OFF + KB * NR * D * 4;      // weights [warps][8 tokens][NR]
  static constexpr int A_OFF = P_OFF + kWarps * 8 * NR * 4;  // rescales [warps][NR]
  static constexpr int BYTES = A_OFF + kWarps * NR * 4;
  static constexpr int RPL = NR < 4 ? 1 : NR / 4;             // rows of a lane, once reduced
  static constexpr int CPL = D / 32, CV = CPL < 4 ? CPL : 4;  // a lane's channels, CV side by side
};

// N = 2 or 4 consecutive stored values as float32.
template <int VK, int N>
I4KV_DEVINL void load_values(const void* base, size_t i, float (&x)[N]) {
  if constexpr (VK == INT4KV_VALUES_F32 && N == 4) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    load_f32<N>(base, VK, i, x);
  }
}

template <bool FIRST, class A, class B>
I4KV_DEVINL auto& pick(A& a, B& b) {
  if constexpr (FIRST) return a;
  else return b;
}

// (s0, s1) += (a0 b0, a1 b1), each rounded once.
I4KV_DEVINL void dot2(float (&s)[2], float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 s, x, y;\n\tmov.b64 s, {%0, %1};\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tfma.rn.f32x2 s, x, y, s;\n\t"
      "mov.b64 {%0, %1}, s;\n\t}"
      : "+f"(s[0]), "+f"(s[1])
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

template <int D, int NR, int VK>
__global__ void __launch_bounds__(kThreads) multi_query_f32_kernel(MultiQueryArgs a) {
  using S = Shape<D, NR, VK>;
  constexpr int TOK = S::TOK, TP = S::TP, RPL = S::RPL, CPL = S::CPL, CV = S::CV;
  extern __shared__ __align__(128) char smem[];
  __shared__ uint64_t s_full[2], s_empty[2];
  __shared__ uint32_t s_pages[2];
  __shared__ RunPlan s_plan;
  __shared__ float s_m[kWarps][NR], s_l[kWarps][NR];
  __shared__ int s_edge[NR], s_depth[kMqMaxDrafts];
  __shared__ uint64_t s_word[NR];
  __shared__ volatile int s_failed;  // a wait ran out: nobody waits any more
  float* s_q = reinterpret_cast<float*>(smem + S::Q_OFF);
  float* s_o = reinterpret_cast<float*>(smem + S::O_OFF);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  grid_dependency_wait();
  allow_dependent_launch();
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], TP);
      mbar_init(&s_empty[i], kWarps);
    }
    s_failed = 0;
    fence_barrier_init();
  }
  zero_idle_rows<NR, TP, D>(a);
  const int cta = blockIdx.x;
  if (warp == 0) {
    const RunPlan mine = plan_run<NR, TP, kStreamUnits, kDraftUnits>(a, cta, gridDim.x);
    if (lane == 0) s_plan = mine;
  }
  __syncthreads();
  const RunPlan plan = s_plan;
  if (tid == 0) a.tails[cta] = RunTail{};  // (overwritten by the same thread where the run shares its last stream)
  if (plan.tiles == 0) return;
  const int u1 = plan.tiles;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_try_wait(bar, parity) && !s_failed && !mbar_wait_bounded(bar, parity, kWaitNs)) {
      s_failed = 1;
      mq_status(a.status, kStatusWaitTimeout);
    }
  };

  SeqWork w = seq_work<NR, TP>(a, plan.b, false);
  TileAt p = tile_at(a, w, plan.b, plan.rem);
  auto step = [&]() {
    if (++p.tile >= w.tiles) next_stream<NR, TP>(a, w, p);
  };

  if (warp == kWarps) {
    // ---- copies: lanes < TP, a page each ----
#pragma unroll 1
    for (int u = 0; u < u1; ++u) {
      const int st = u & 1;
      // (the pages are looked up while the stage is still in use)
      uint32_t bytes = 0;
      int phys = 0, home = 0, rows = 0;
      bool ok = false;
      if (lane < TP) {
        const int pg = tile_page<TP>(w, p.tile, lane);
        if (p.tile < w.cache_tiles && page_visible(w, pg)) {
          const int32_t* bt = a.block_table + (size_t)p.b * a.max_pages;
          phys = __ldg(bt + pg);
          home = __ldg(bt + pg / a.group_pages * a.group_pages);
          rows = min(kMqPage, w.len - pg * kMqPage);
          ok = phys >= 0 && phys < a.num_pages && home >= 0 && home < a.num_pages;
          if (!ok) mq_status(a.status, kStatusBadPage);
          if (ok) bytes = (uint32_t)rows * (D * S::VB + D / 2) + 2 * D * 4;
        }
      }
      const uint32_t live = __ballot_sync(0xffffffffu, ok);
      wait(&s_empty[st], (uint32_t)((u >> 1) + 1) & 1);
      __syncwarp();
      if (s_failed) {  // the copies issued so far land, or a bound passes
        for (int v = max(0, u - 2); v < u; ++v) mbar_wait_bounded(&s_full[v & 1], (uint32_t)(v >> 1) & 1, 10000000ull);
        break;
      }
      if (lane == 0) s_pages[st] = live;
      __syncwarp();
      if (lane < TP) mbar_arrive_expect_tx(&s_full[st], bytes);
      if (ok) {
        char* base = smem + st * S::STAGE;
        const size_t slab = ((size_t)phys * a.kv_heads + p.head) * kMqPage;
        bulk_g2s(base + S::V_BYTES + lane * kMqPage * D / 2, a.k_pool + slab * (D / 2), (uint32_t)rows * (D / 2),
                 &s_full[st]);
        bulk_g2s(base + S::V_BYTES + S::K_BYTES + lane * 2 * D * 4,
                 a.sz_pool + ((size_t)home * a.kv_heads + p.head) * 2 * D, 2 * D * 4, &s_full[st]);
        bulk_g2s(base + lane * kMqPage * D * S::VB, static_cast<const char*>(a.v_pool) + slab * D * S::VB,
                 (uint32_t)rows * D * S::VB, &s_full[st]);
      }
      step();
    }
    return;
  }

  const int ql = lane & 7, tl = lane >> 3;        // logits: channels 8 ql + 64 i of tokens tl, tl + 4
  const int swap = ql & 4;                        // these lanes' second quad of channels comes first
  const int my_tok = tl + 4 * (ql >> 2);          // after the reduction: this token of the warp's 8,
  const int my_row = (ql & 3) * (NR < 4 ? 0 : RPL);  // rows my_row + j
  float* s_p = reinterpret_cast<float*>(smem + S::P_OFF) + warp * 8 * NR;
  float* s_al = reinterpret_cast<float*>(smem + S::A_OFF) + warp * NR;
  float m_run[RPL], l_run[RPL];  // maxima; this lane's share of the sums
  float acc[NR][CPL];
  bool fresh = true;

#pragma unroll 1
  for (int u = 0; u < u1; ++u) {
    const int st = u & 1;
    if (fresh) {  // a stream begins (no warp is in another tile): its queries and what they see
      fresh = false;
#pragma unroll
      for (int j = 0; j < RPL; ++j) {
        m_run[j] = -INFINITY;
        l_run[j] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int c = 0; c < CPL; ++c) acc[r][c] = 0.f;
      for (int i = 2 * tid; i < NR * D; i += 2 * kConsumers) {
        const int r = i / D, rr = p.chunk * NR + r;
        float x[2] = {0.f, 0.f};
        if (rr < w.rows) load_f32<2>(a.q, a.qk, row_offset(a, w, p.head, rr, D) + (i - r * D), x);
        s_q[i] = x[0];
        s_q[i + 1] = x[1];
      }
      if (tid < NR) {
        const int rr = p.chunk * NR + tid, t = min(rr, w.rows - 1) / a.group_q;
        uint64_t word = 0;
        if (a.mask) word = (uint64_t)a.mask[w.row0 + t];
        s_word[tid] = word;
        s_edge[tid] = a.window > 0 ? w.pos0 + (a.mask ? draft_depth(word, t, w.drafts) : 0) - a.window : -1;
      }
      if (a.mask && tid < w.drafts) s_depth[tid] = draft_depth((uint64_t)a.mask[w.row0 + tid], tid, w.drafts);
      named_bar_sync(1, kConsumers);
    }
    const bool in_cache = p.tile < w.cache_tiles;
    wait(&s_full[st], (uint32_t)(u >> 1) & 1);
    const char* base = smem + st * S::STAGE;
    const int tok0 = warp * 8;  // the warp's tokens: half a page
    const int pos0 = in_cache ? tile_page<TP>(w, p.tile, tok0 / kMqPage) * kMqPage + tok0 % kMqPage
                              : (p.tile - w.cache_tiles) * TOK + tok0;  // position, or draft, of the first
    const int there = in_cache ? ((s_pages[st] >> (tok0 / kMqPage) & 1) ? min(8, w.len - pos0) : 0)
                               : min(8, w.drafts - pos0);
    if (there > 0) {
      // ---- logits ----
      float x[RPL];
      {
        float s2[2][NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) s2[0][r][0] = s2[0][r][1] = s2[1][r][0] = s2[1][r][1] = 0.f;
#pragma unroll(NR <= 4 ? 2 : 1)
        for (int c = 8 * ql; c < D; c += 64) {
          float k[2][8];
          if (in_cache) {  // (rows behind the length hold what the stage held: never used)
            const char* krow = base + S::V_BYTES + (tok0 + tl) * (D / 2) + c / 2;
            const float* sz = reinterpret_cast<const float*>(base + S::V_BYTES + S::K_BYTES) + tok0 / kMqPage * 2 * D + c;
            uint32_t w0 = *reinterpret_cast<const uint32_t*>(krow), w1 = *reinterpret_cast<const uint32_t*>(krow + 2 * D);
            w0 = __funnelshift_r(w0, w0, 4 * swap);
            w1 = __funnelshift_r(w1, w1, 4 * swap);
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
              const float4 sc = *reinterpret_cast<const float4*>(sz + (j ^ swap));
              const float4 zp = *reinterpret_cast<const float4*>(sz + D + (j ^ swap));
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t wd = e ? w1 : w0;
                k[e][j] = ((float)((wd >> (4 * j)) & 15u) - zp.x) * sc.x;
                k[e][j + 1] = ((float)((wd >> (4 * j + 4)) & 15u) - zp.y) * sc.y;
                k[e][j + 2] = ((float)((wd >> (4 * j + 8)) & 15u) - zp.z) * sc.z;
                k[e][j + 3] = ((float)((wd >> (4 * j + 12)) & 15u) - zp.w) * sc.w;
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int j = 0; j < 8; ++j) k[e][j] = 0.f;
              if (tl + 4 * e < there) {
                const size_t row = ((size_t)(w.row0 + pos0 + tl + 4 * e) * a.kv_heads + p.head) * D + c;
                float y[4];
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                  load_f32<4>(a.kd, a.qk, row + (j ^ swap), y);
                  k[e][j] = y[0]; k[e][j + 1] = y[1]; k[e][j + 2] = y[2]; k[e][j + 3] = y[3];
                }
              }
            }
          }
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float4 y0 = *reinterpret_cast<const float4*>(s_q + r * D + c + swap);
            const float4 y1 = *reinterpret_cast<const float4*>(s_q + r * D + c + (4 ^ swap));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              dot2(s2[e][r], k[e][0], k[e][1], y0.x, y0.y);
              dot2(s2[e][r], k[e][2], k[e][3], y0.z, y0.w);
              dot2(s2[e][r], k[e][4], k[e][5], y1.x, y1.y);
              dot2(s2[e][r], k[e][6], k[e][7], y1.z, y1.w);
            }
          }
        }
        // reduce-scatter over the 8 lanes of a token: token tl + 4 to the upper four,
        // then quarters of the rows
        float v[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float x0 = s2[0][r][0] + s2[0][r][1], x1 = s2[1][r][0] + s2[1][r][1];
          const float give = ql & 4 ? x0 : x1, keep = ql & 4 ? x1 : x0;
          v[r] = keep + __shfl_xor_sync(0xffffffffu, give, 4);
        }
        if constexpr (NR == 1) {
          v[0] += __shfl_xor_sync(0xffffffffu, v[0], 2);
          v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1);
          x[0] = v[0];
        } else {
          float v2[NR / 2];
#pragma unroll
          for (int r = 0; r < NR / 2; ++r) {
            const float give = ql & 2 ? v[r] : v[r + NR / 2], keep = ql & 2 ? v[r + NR / 2] : v[r];
            v2[r] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
          }
#pragma unroll
          for (int r = 0; r < RPL; ++r) {
            const float give = ql & 1 ? v2[r] : v2[r + RPL], keep = ql & 1 ? v2[r + RPL] : v2[r];
            x[r] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
          }
        }
      }
      // ---- what the rows see ----
      const int at = pos0 + my_tok;
      const bool real = my_tok < there;
      bool guard = !real;
      if (!in_cache || a.window > 0) {
        const int behind = in_cache ? at : (real && a.window > 0 ? w.pos0 + s_depth[at] : 0);
#pragma unroll
        for (int j = 0; j < RPL; ++j) {
          const int r = my_row + j;
          bool sees = in_cache || (s_word[r] >> (at & 63) & 1);
          if (a.window > 0) sees = sees && (behind > s_edge[r] || behind < a.sinks);
          guard = guard || !sees;
          if (!sees) x[j] = -INFINITY;
        }
      }
      if (!real) {
#pragma unroll
        for (int j = 0; j < RPL; ++j) x[j] = -INFINITY;
      }
      guard = __any_sync(0xffffffffu, guard);
      // ---- softmax over the warp's 8 tokens ----
#pragma unroll
      for (int j = 0; j < RPL; ++j) {
        float mx = fmaxf(m_run[j], x[j]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float al = mx == -INFINITY ? 1.f : exp2_fast((m_run[j] - mx) * kLog2e);
        const float e = x[j] == -INFINITY ? 0.f : exp2_fast((x[j] - mx) * kLog2e);
        l_run[j] = fmaf(l_run[j], al, e);
        m_run[j] = mx;
        const int r = my_row + j;
        if (NR >= 4 || (ql & 3) == 0) s_p[my_tok * NR + r] = e;
        if (lane < 4 && (NR >= 4 || lane == 0)) s_al[r] = al;
      }
      __syncwarp();
      // ---- values: the tile's sum from zero, then added to the running one (a
      // shorter chain of roundings); with many sums straight into those ----
      constexpr bool kApart = NR * CPL < 64;
      float sum[kApart ? NR : 1][kApart ? CPL : 1];
      auto& ps = pick<kApart>(sum, acc);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float al = kApart ? 0.f : s_al[r];
#pragma unroll
        for (int c = 0; c < CPL; ++c) ps[r][c] = kApart ? 0.f : ps[r][c] * al;
      }
      auto value = [&](int t, int c0, float (&v)[CV]) {
        const int ch = c0 / CV * 32 * CV + lane * CV;
        if (in_cache) load_values<VK, CV>(base, (size_t)(tok0 + t) * D + ch, v);
        else load_f32<CV>(a.vd, a.qk, ((size_t)(w.row0 + pos0 + t) * a.kv_heads + p.head) * D + ch, v);
      };
      if (!guard) {
#pragma unroll 4
        for (int t = 0; t < 8; ++t) {
#pragma unroll
          for (int c0 = 0; c0 < CPL; c0 += CV) {
            float v[CV];
            value(t, c0, v);
            if constexpr (NR == 1) {
#pragma unroll
              for (int c = 0; c < CV; c += 2) fma2_rn(ps[0][c0 + c], ps[0][c0 + c + 1], v[c], v[c + 1], s_p[t]);
            } else {  // pairs of rows
#pragma unroll
              for (int r = 0; r < NR; r += 4) {
                const float4 e = *reinterpret_cast<const float4*>(s_p + t * NR + r);
#pragma unroll
                for (int c = 0; c < CV; ++c) {
                  fma2_rn(ps[r][c0 + c], ps[r + 1][c0 + c], e.x, e.y, v[c]);
                  fma2_rn(ps[r + 2][c0 + c], ps[r + 3][c0 + c], e.z, e.w, v[c]);
                }
              }
            }
          }
        }
      } else {  // some row does not see some token: what stands there, even NaN, adds nothing
#pragma unroll 1
        for (int t = 0; t < there; ++t) {
#pragma unroll
          for (int c0 = 0; c0 < CPL; c0 += CV) {
            float v[CV];
            value(t, c0, v);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              const float e = s_p[t * NR + r];
              if (e != 0.f) {
#pragma unroll
                for (int c = 0; c < CV; c += 2) fma2_rn(ps[r][c0 + c], ps[r][c0 + c + 1], v[c], v[c + 1], e);
              }
            }
          }
        }
      }
      if constexpr (kApart) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float al = s_al[r];
#pragma unroll
          for (int c = 0; c < CPL; ++c) acc[r][c] = fmaf(acc[r][c], al, sum[r][c]);
        }
      }
    }
    __syncwarp();  // (the weights and the stage are free)
    if (lane == 0) mbar_arrive(&s_empty[st]);

    // ---- the stream, or this run's share of it, ends: the warps meet ----
    const bool ends = p.tile + 1 >= w.tiles;
    if (ends || u + 1 == u1) {
#pragma unroll
      for (int j = 0; j < RPL; ++j) {
        float l = l_run[j];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane < 4 && (NR >= 4 || lane == 0)) {
          s_m[warp][my_row + j] = m_run[j];
          s_l[warp][my_row + j] = l;
        }
      }
      named_bar_sync(1, kConsumers);
      auto top_of = [&](int r) {
        float m = s_m[0][r];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) m = fmaxf(m, s_m[i][r]);
        return m;
      };
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float m = top_of(r), al = m == -INFINITY ? 1.f : exp2_fast((s_m[warp][r] - m) * kLog2e);
#pragma unroll
        for (int c = 0; c < CPL; ++c) acc[r][c] *= al;
      }
#pragma unroll 1
      for (int turn = 0; turn < kWarps / S::KB; ++turn) {
        if (warp / S::KB == turn) {
          float* o = s_o + warp % S::KB * (NR * D);
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int c = 0; c < CPL; ++c) {
              float* at = o + r * D + c / CV * 32 * CV + lane * CV + c % CV;
              *at = turn == 0 ? acc[r][c] : *at + acc[r][c];
            }
        }
        named_bar_sync(1, kConsumers);
      }
      const int first = u - p.tile;  // the stream's first tile
      const bool whole = ends && first >= 0;
      float* rec = a.recs + (size_t)(2 * cta + (first > 0 ? 1 : 0)) * Record<NR, D>::kFloats;
      for (int i = 2 * tid; i < NR * D; i += 2 * kConsumers) {
        const int r = i / D, c = i - r * D, rr = p.chunk * NR + r;
        if (rr >= w.rows) continue;
        float2 y = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < S::KB; ++k) {
          const float2 z = *reinterpret_cast<const float2*>(s_o + k * (NR * D) + i);
          y.x += z.x;
          y.y += z.y;
        }
        const float m = top_of(r);
        float l = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) l += m == -INFINITY ? 0.f : s_l[k][r] * exp2_fast((s_m[k][r] - m) * kLog2e);
        if (whole) {
          const float inv = 1.f / fmaxf(l, 1e-10f);
          store2(a.out, a.qk, row_offset(a, w, p.head, rr, D) + c, y.x * inv, y.y * inv);
        } else {
          *reinterpret_cast<float2*>(rec + 2 * NR + i) = y;
          if (c == 0) {
            rec[r] = m;
            rec[NR + r] = l;
          }
        }
      }
      fresh = true;
      if (u + 1 == u1 && tid == 0) note_tail(a, cta, plan, w, p, NR);
      named_bar_sync(1, kConsumers);  // (s_o, s_m and s_l are free)
    }
    step();
  }
}

template <int D, int NR, int VK>
cudaError_t launch(const MultiQueryArgs& args, int sms, void* ws, size_t ws_bytes, cudaStream_t stream) {
  using S = Shape<D, NR, VK>;
  constexpr auto kern = multi_query_f32_kernel<D, NR, VK>;
  static_assert(S::BYTES <= 225 * 1024, "shared memory");
  int per_sm = 0;
  cudaError_t e = mq_occupancy<kern>(kThreads, S::BYTES, &per_sm);
  if (e != cudaSuccess) return e;
  const int runs = sms * std::min(per_sm, kMaxPerSm);
  MultiQueryArgs a = args;
  if (!mq_workspace(a, ws, ws_bytes, runs, Record<NR, D>::kFloats)) return cudaErrorInvalidValue;
  e = mq_launch_pdl(kern, dim3(runs), dim3(kThreads), S::BYTES, stream, a);
  if (e != cudaSuccess) return e;
  return mq_launch_pdl(merge_records_kernel<NR, D>, dim3(runs - 1, (NR + kMergeWarps - 1) / kMergeWarps),
                       dim3(kMergeWarps * 32), 0, stream, a);
}

template <int D, int NR>
cudaError_t launch_vk(int vk, const MultiQueryArgs& a, int sms, void* ws, size_t n, cudaStream_t st) {
  if (vk == INT4KV_VALUES_F32) return launch<D, NR, INT4KV_VALUES_F32>(a, sms, ws, n, st);
  if (vk == INT4KV_VALUES_F16) return launch<D, NR, INT4KV_VALUES_F16>(a, sms, ws, n, st);
  return launch<D, NR, INT4KV_VALUES_BF16>(a, sms, ws, n, st);
}

// Rows of a chunk.
int chunk_of(long long rows, int dim) { return rows == 1 ? 1 : (rows <= 4 ? 4 : (rows <= 8 || dim == 256 ? 8 : 16)); }
long long rows_of(const MultiQueryArgs& a) { return (long long)std::max(1, a.max_drafts) * a.group_q; }

template <int D>
cudaError_t launch_rows(int nr, int vk, const MultiQueryArgs& a, int sms, void* ws, size_t n, cudaStream_t st) {
  if (nr == 1) return launch_vk<D, 1>(vk, a, sms, ws, n, st);
  if (nr == 4) return launch_vk<D, 4>(vk, a, sms, ws, n, st);
  if constexpr (D < 256) {
    if (nr == 16) return launch_vk<D, 16>(vk, a, sms, ws, n, st);
  }
  return launch_vk<D, 8>(vk, a, sms, ws, n, st);
}

}  // namespace

namespace i4kv {

double multi_query_f32_units(const MultiQueryArgs& a, int dim) {
  return mq_most_units(a, rows_of(a), chunk_of(rows_of(a), dim), 64 / kMqPage, kStreamUnits + kDraftUnits);
}

size_t multi_query_f32_workspace(int dim, int sms) {
  return mq_workspace_bytes(sms * kMaxPerSm, 2 * 16 + 16 * dim);
}

cudaError_t multi_query_f32(const MultiQueryArgs& a, int dim, int vk, int sms, void* ws, size_t ws_bytes,
                            cudaStream_t stream) {
  const int nr = chunk_of(rows_of(a), dim);
  if (dim == 64) return launch_rows<64>(nr, vk, a, sms, ws, ws_bytes, stream);
  if (dim == 128) return launch_rows<128>(nr, vk, a, sms, ws, ws_bytes, stream);
  return launch_rows<256>(nr, vk, a, sms, ws, ws_bytes, stream);
}

}  // namespace i4kv
