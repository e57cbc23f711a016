// Several queries of a sequence over its paged INT4 cache in float32: drafted
// trees (int4kv_paged_tree_decode) and sliding windows with sinks
// (int4kv_paged_window_decode).
//
// Math: per row, logits x_j = sum_c q_c (code_jc s_c - zp_c s_c) over the
// visible cached tokens and q . k over the visible drafts, one pass with the
// running maximum m and sum l, out = sum_j 2^((x_j - m) log2 e) v_j / l. Keys
// are dequantized in registers, once for the NR rows of a CTA; products and
// sums are float32 in paired instructions (two lanes of work per issue). A
// tile's values are summed from zero and then added to the running sum, so a
// long cache costs two short sums instead of one long one: the error stays
// near 2^-24 sqrt(tokens / TOK) instead of 2^-24 sqrt(tokens).
//
// Layout of the work in a CTA of eight warps over a tile of TOK tokens:
//   logits: a lane holds one token and 8 of every 32 channels (word lane & 3 of
//     each 16 bytes of the packed row), so code words, scales and queries are
//     read from shared memory without bank conflicts, and two shuffles finish a
//     logit; every row reuses the dequantized channels from registers.
//   softmax: a warp a row, lanes over the tokens.
//   values: a thread holds two channels of all NR rows and a share of the tile's
//     tokens; the shares meet in shared memory when the stream ends.
// Pages arrive by bulk copies into a two-stage ring, the next tile's while the
// current one is computed. Which of bytes and arithmetic bounds it depends on
// NR: a tile costs NR * 2 * D * TOK fused multiply-adds whatever the rows'
// count, so NR is the smallest of 1, 4, 8, 16 that holds the rows of one kv head.
#include <algorithm>

#include "multi_query.cuh"

using namespace i4kv;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPerSm = 4;                  // CTAs per SM the workspace is sized for
constexpr uint64_t kWaitNs = 2000000000ull;  // bounded waits: 2 s

template <int D, int NR, int VK>
struct Shape {
  static constexpr int TOK = D == 256 ? 32 : 64;
  static constexpr int TP = TOK / kMqPage;
  static constexpr int VB = VK == INT4KV_VALUES_F32 ? 4 : 2;
  static constexpr int V_BYTES = TOK * D * VB, K_BYTES = TOK * D / 2, SZ_BYTES = TP * 2 * D * 4;
  static constexpr int STAGE = V_BYTES + K_BYTES + SZ_BYTES;
  static constexpr int P_STRIDE = NR == 1 ? 1 : NR + 4;
  static constexpr int Q_OFF = 2 * STAGE;
  static constexpr int O_OFF = Q_OFF + NR * D * 4;
  static constexpr int S_OFF = O_OFF + NR * D * 4;
  static constexpr int P_OFF = S_OFF + NR * (TOK + 4) * 4;  // (16-byte aligned: TOK is a multiple of 4)
  static constexpr int BYTES = P_OFF + TOK * P_STRIDE * 4;
  static constexpr int PAIRS = D / 2, TG = kThreads / PAIRS, TPG = TOK / TG;
};

template <int D, int NR, int VK>
__global__ void __launch_bounds__(kThreads) multi_query_f32_kernel(MultiQueryArgs a) {
  using S = Shape<D, NR, VK>;
  constexpr int TOK = S::TOK, TP = S::TP;
  extern __shared__ __align__(128) char smem[];
  __shared__ uint64_t s_full[2];
  __shared__ uint32_t s_pages[2];
  __shared__ RunPlan s_plan;
  __shared__ float s_alpha[NR], s_m[NR], s_l[NR];
  __shared__ int s_edge[NR], s_depth[kMqMaxDrafts];
  __shared__ uint64_t s_word[NR];
  float* s_q = reinterpret_cast<float*>(smem + S::Q_OFF);
  float* s_o = reinterpret_cast<float*>(smem + S::O_OFF);
  float* s_s = reinterpret_cast<float*>(smem + S::S_OFF);
  float* s_p = reinterpret_cast<float*>(smem + S::P_OFF);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  grid_dependency_wait();
  allow_dependent_launch();
  if (tid == 0) {
    mbar_init(&s_full[0], TP);
    mbar_init(&s_full[1], TP);
    fence_barrier_init();
  }
  zero_idle_rows<NR, TP, D>(a);
  const int cta = blockIdx.x;
  if (warp == 0) {
    const RunPlan mine = plan_run<NR, TP, 1, 1>(a, cta, gridDim.x);
    if (lane == 0) s_plan = mine;
  }
  __syncthreads();
  const RunPlan plan = s_plan;
  if (plan.tiles == 0) {
    if (tid == 0) a.tails[cta] = RunTail{};
    return;
  }
  const int u1 = plan.tiles;

  SeqWork w = seq_work<NR, TP>(a, plan.b, false), nw = w;  // of the current tile, of the next copied one
  TileAt p = tile_at(a, w, plan.b, plan.rem), np = p;

  // Copies of tile `np` into stage st (lanes < TP of warp 0, a page each).
  auto issue = [&](int st) {
    if (lane < TP) {
      uint32_t bytes = 0;
      int phys = 0, home = 0, rows = 0;
      bool ok = false;
      const int pg = tile_page<TP>(nw, np.tile, lane);
      if (np.tile < nw.cache_tiles && page_visible(nw, pg)) {
        const int32_t* bt = a.block_table + (size_t)np.b * a.max_pages;
        phys = __ldg(bt + pg);
        home = __ldg(bt + pg / a.group_pages * a.group_pages);
        rows = min(kMqPage, nw.len - pg * kMqPage);
        ok = phys >= 0 && phys < a.num_pages && home >= 0 && home < a.num_pages;
        if (!ok) mq_status(a.status, kStatusBadPage);
        if (ok) bytes = (uint32_t)rows * (D * S::VB + D / 2) + 2 * D * 4;
      }
      const uint32_t live = __ballot_sync((1u << TP) - 1, ok);
      if (lane == 0) s_pages[st] = live;
      __syncwarp((1u << TP) - 1);
      fence_proxy_async_smem();
      mbar_arrive_expect_tx(&s_full[st], bytes);
      if (ok) {
        char* base = smem + st * S::STAGE;
        const size_t slab = ((size_t)phys * a.kv_heads + np.head) * kMqPage;
        bulk_g2s(base + lane * kMqPage * D * S::VB, static_cast<const char*>(a.v_pool) + slab * D * S::VB,
                 (uint32_t)rows * D * S::VB, &s_full[st]);
        bulk_g2s(base + S::V_BYTES + lane * kMqPage * D / 2, a.k_pool + slab * (D / 2),
                 (uint32_t)rows * (D / 2), &s_full[st]);
        bulk_g2s(base + S::V_BYTES + S::K_BYTES + lane * 2 * D * 4,
                 a.sz_pool + ((size_t)home * a.kv_heads + np.head) * 2 * D, 2 * D * 4, &s_full[st]);
      }
    }
  };
  auto step = [&](SeqWork& sw, TileAt& t) {
    if (++t.tile >= sw.tiles) next_stream<NR, TP>(a, sw, t);
  };

  constexpr int RPW = (NR + 7) / 8;  // softmax rows of a warp: warp, warp + 8
  float m_run[RPW], l_run[RPW];
  float acc[NR][2];
  const int pair = tid % S::PAIRS, group = tid / S::PAIRS;

  if (warp == 0) issue(0);
  step(nw, np);
  int copied = 1;
  bool fresh = true;

  for (int u = 0; u < u1; ++u) {
    const int st = u & 1;
    const uint32_t parity = (uint32_t)((u >> 1) & 1);
    __syncthreads();  // everyone is done with the previous tile
    if (copied < u1) {
      if (warp == 0) issue(st ^ 1);
      if (++copied < u1) step(nw, np);
    }
    if (fresh) {  // a stream begins: its queries and what they see
      fresh = false;
#pragma unroll
      for (int j = 0; j < RPW; ++j) {
        m_run[j] = -INFINITY;
        l_run[j] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) acc[r][0] = acc[r][1] = 0.f;
      for (int i = 2 * tid; i < NR * D; i += 2 * kThreads) {
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
      __syncthreads();
    }
    const bool in_cache = p.tile < w.cache_tiles;
    if (in_cache) {
      if (!mbar_wait_bounded(&s_full[st], parity, kWaitNs)) mq_status(a.status, kStatusWaitTimeout);
    } else {
      mbar_wait_bounded(&s_full[st], parity, kWaitNs);  // an empty phase
    }
    const char* base = smem + st * S::STAGE;

    // ---- logits ----
    constexpr int kPasses = TOK / 64 == 0 ? 1 : TOK / 64;  // 8 warps x 8 tokens
    bool all_seen = true;
#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) {
      const int tok = ps * 64 + warp * 8 + (lane >> 2), qd = lane & 3;
      if (tok < TOK) {
        float s2[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) s2[r][0] = s2[r][1] = 0.f;
        auto rows_add = [&](const float (&k)[8], int c) {
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float4 x = *reinterpret_cast<const float4*>(s_q + r * D + c);
            const float4 y = *reinterpret_cast<const float4*>(s_q + r * D + c + 4);
            asm("{\n\t.reg .b64 s, x, y;\n\tmov.b64 s, {%0, %1};\n\t"
                "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tfma.rn.f32x2 s, x, y, s;\n\t"
                "mov.b64 {%0, %1}, s;\n\t}"
                : "+f"(s2[r][0]), "+f"(s2[r][1]) : "f"(k[0]), "f"(k[1]), "f"(x.x), "f"(x.y));
            asm("{\n\t.reg .b64 s, x, y;\n\tmov.b64 s, {%0, %1};\n\t"
                "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tfma.rn.f32x2 s, x, y, s;\n\t"
                "mov.b64 {%0, %1}, s;\n\t}"
                : "+f"(s2[r][0]), "+f"(s2[r][1]) : "f"(k[2]), "f"(k[3]), "f"(x.z), "f"(x.w));
            asm("{\n\t.reg .b64 s, x, y;\n\tmov.b64 s, {%0, %1};\n\t"
                "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tfma.rn.f32x2 s, x, y, s;\n\t"
                "mov.b64 {%0, %1}, s;\n\t}"
                : "+f"(s2[r][0]), "+f"(s2[r][1]) : "f"(k[4]), "f"(k[5]), "f"(y.x), "f"(y.y));
            asm("{\n\t.reg .b64 s, x, y;\n\tmov.b64 s, {%0, %1};\n\t"
                "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tfma.rn.f32x2 s, x, y, s;\n\t"
                "mov.b64 {%0, %1}, s;\n\t}"
                : "+f"(s2[r][0]), "+f"(s2[r][1]) : "f"(k[6]), "f"(k[7]), "f"(y.z), "f"(y.w));
          }
        };
        int at;        // position of the token (cache), or index of the draft
        bool real;
        if (in_cache) {
          at = tile_page<TP>(w, p.tile, tok / kMqPage) * kMqPage + tok % kMqPage;
          real = at < w.len && (s_pages[st] >> (tok / kMqPage) & 1);
          const char* krow = base + S::V_BYTES + tok * (D / 2);
          const float* sz = reinterpret_cast<const float*>(base + S::V_BYTES + S::K_BYTES) + tok / kMqPage * 2 * D;
          if (real) {
#pragma unroll 2
            for (int c = 8 * qd; c < D; c += 32) {
              const uint32_t wd = *reinterpret_cast<const uint32_t*>(krow + c / 2);
              float k[8];
#pragma unroll
              for (int j = 0; j < 8; j += 4) {
                const float4 sc = *reinterpret_cast<const float4*>(sz + c + j);
                const float4 zp = *reinterpret_cast<const float4*>(sz + D + c + j);
                k[j] = ((float)((wd >> (4 * j)) & 15u) - zp.x) * sc.x;
                k[j + 1] = ((float)((wd >> (4 * j + 4)) & 15u) - zp.y) * sc.y;
                k[j + 2] = ((float)((wd >> (4 * j + 8)) & 15u) - zp.z) * sc.z;
                k[j + 3] = ((float)((wd >> (4 * j + 12)) & 15u) - zp.w) * sc.w;
              }
              rows_add(k, c);
            }
          }
        } else {
          at = (p.tile - w.cache_tiles) * TOK + tok;
          real = at < w.drafts;
          if (real) {
            const size_t row = ((size_t)(w.row0 + at) * a.kv_heads + p.head) * D;
            for (int c = 8 * qd; c < D; c += 32) {
              float k[8];
              load_f32<8>(a.kd, a.qk, row + c, k);
              rows_add(k, c);
            }
          }
        }
        float mine[(NR + 3) / 4] = {};
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float x = s2[r][0] + s2[r][1];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if ((r & 3) == qd) mine[r >> 2] = x;
        }
        const int behind = in_cache ? at : (real && a.window > 0 ? w.pos0 + s_depth[at] : 0);
#pragma unroll
        for (int j = 0; j < (NR + 3) / 4; ++j) {
          const int r = 4 * j + qd;
          if (NR == 1 && qd != 0) break;
          bool sees = real;
          if (!in_cache) sees = sees && (s_word[r] >> (at & 63) & 1);
          if (a.window > 0) sees = sees && (behind > s_edge[r] || behind < a.sinks);
          all_seen = all_seen && sees;
          s_s[r * (TOK + 4) + tok] = sees ? mine[j] : -INFINITY;
        }
      }
    }
    const bool guard = !__syncthreads_and(all_seen);

    // ---- softmax: warp w has rows w, w + 8 ----
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
      const int r = warp + 8 * j;
      if (r < NR) {
        float x[TOK / 32];
        float mx = m_run[j];
#pragma unroll
        for (int i = 0; i < TOK / 32; ++i) {
          x[i] = s_s[r * (TOK + 4) + 32 * i + lane];
          mx = fmaxf(mx, x[i]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float al = mx == -INFINITY ? 1.f : exp2_fast((m_run[j] - mx) * kLog2e);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < TOK / 32; ++i) {
          const float e = x[i] == -INFINITY ? 0.f : exp2_fast((x[i] - mx) * kLog2e);
          s_p[(32 * i + lane) * S::P_STRIDE + r] = e;
          sum += e;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l_run[j] = fmaf(l_run[j], al, sum);
        m_run[j] = mx;
        if (lane == 0) s_alpha[r] = al;
      }
    }
    __syncthreads();

    // ---- values ----
    {
      float ps[NR][2];
#pragma unroll
      for (int r = 0; r < NR; ++r) ps[r][0] = ps[r][1] = 0.f;
      const int t0 = group * S::TPG;
      auto value = [&](int t, float (&v)[2]) {
        if (in_cache) {
          load_f32<2>(base, VK, (size_t)t * D + 2 * pair, v);
        } else {
          const int at = (p.tile - w.cache_tiles) * TOK + t;
          v[0] = v[1] = 0.f;
          if (at < w.drafts)
            load_f32<2>(a.vd, a.qk, ((size_t)(w.row0 + at) * a.kv_heads + p.head) * D + 2 * pair, v);
        }
      };
      if (!guard) {
#pragma unroll 4
        for (int t = t0; t < t0 + S::TPG; ++t) {
          float v[2];
          value(t, v);
          if (NR == 1) fma2_rn(ps[0][0], ps[0][1], v[0], v[1], s_p[t]);
#pragma unroll
          for (int r = 0; r + 4 <= NR; r += 4) {
            const float4 e = *reinterpret_cast<const float4*>(s_p + t * S::P_STRIDE + r);
            fma2_rn(ps[r][0], ps[r][1], v[0], v[1], e.x);
            fma2_rn(ps[r + 1][0], ps[r + 1][1], v[0], v[1], e.y);
            fma2_rn(ps[r + 2][0], ps[r + 2][1], v[0], v[1], e.z);
            fma2_rn(ps[r + 3][0], ps[r + 3][1], v[0], v[1], e.w);
          }
        }
      } else {  // some row does not see some token: what stands there, even NaN, adds nothing
        static_assert(S::TPG % 4 == 0, "four tokens a turn");
#pragma unroll 1
        for (int t4 = t0; t4 < t0 + S::TPG; t4 += 4) {
          float v[4][2];
#pragma unroll
          for (int t = 0; t < 4; ++t) value(t4 + t, v[t]);
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              const float e = s_p[(t4 + t) * S::P_STRIDE + r];
              if (e != 0.f) fma2_rn(ps[r][0], ps[r][1], v[t][0], v[t][1], e);
            }
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float al = s_alpha[r];
        acc[r][0] = fmaf(acc[r][0], al, ps[r][0]);
        acc[r][1] = fmaf(acc[r][1], al, ps[r][1]);
      }
    }

    // ---- the stream, or this run's share of it, ends ----
    const bool ends = p.tile + 1 >= w.tiles;
    if (ends || u + 1 == u1) {
#pragma unroll
      for (int j = 0; j < RPW; ++j) {
        const int r = warp + 8 * j;
        if (r < NR && lane == 0) {
          s_m[r] = m_run[j];
          s_l[r] = l_run[j];
        }
      }
      for (int g = 0; g < S::TG; ++g) {
        if (group == g) {
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float2* o = reinterpret_cast<float2*>(s_o + r * D + 2 * pair);
            float2 x = g == 0 ? make_float2(0.f, 0.f) : *o;
            x.x += acc[r][0];
            x.y += acc[r][1];
            *o = x;
          }
        }
        __syncthreads();
      }
      const int first = u - p.tile;  // the stream's first tile
      const bool whole = ends && first >= 0;
      float* rec = a.recs + (size_t)(2 * cta + (first > 0 ? 1 : 0)) *Record<NR, D>::kFloats;
      for (int i = 2 * tid; i < NR * D; i += 2 * kThreads) {
        const int r = i / D, c = i - r * D, rr = p.chunk * NR + r;
        if (rr >= w.rows) continue;
        const float2 x = *reinterpret_cast<const float2*>(s_o + i);
        if (whole) {
          const float inv = 1.f / fmaxf(s_l[r], 1e-10f);
          store2(a.out, a.qk, row_offset(a, w, p.head, rr, D) + c, x.x * inv, x.y * inv);
        } else {
          *reinterpret_cast<float2*>(rec + 2 * NR + i) = x;
          if (c == 0) {
            rec[r] = s_m[r];
            rec[NR + r] = s_l[r];
          }
        }
      }
      fresh = true;
      if (u + 1 == u1 && tid == 0) note_tail(a, cta, plan, w, p, NR);
    }
    step(w, p);
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

template <int D>
cudaError_t launch_rows(int rows, int vk, const MultiQueryArgs& a, int sms, void* ws, size_t n, cudaStream_t st) {
  if (rows == 1) return launch_vk<D, 1>(vk, a, sms, ws, n, st);
  if (rows <= 4) return launch_vk<D, 4>(vk, a, sms, ws, n, st);
  if (rows <= 8) return launch_vk<D, 8>(vk, a, sms, ws, n, st);
  return launch_vk<D, 16>(vk, a, sms, ws, n, st);
}

}  // namespace

namespace i4kv {

size_t multi_query_f32_workspace(int dim, int sms) {
  return mq_workspace_bytes(sms * kMaxPerSm, 2 * 16 + 16 * dim);
}

cudaError_t multi_query_f32(const MultiQueryArgs& a, int dim, int vk, int sms, void* ws, size_t ws_bytes,
                            cudaStream_t stream) {
  const long long rows = (long long)std::max(1, a.max_drafts) * a.group_q;
  const int r = (int)std::min<long long>(rows, 1 << 20);
  if (dim == 64) return launch_rows<64>(r, vk, a, sms, ws, ws_bytes, stream);
  if (dim == 128) return launch_rows<128>(r, vk, a, sms, ws, ws_bytes, stream);
  return launch_rows<256>(r, vk, a, sms, ws, ws_bytes, stream);
}

}  // namespace i4kv
