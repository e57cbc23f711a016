// Reading a range of tokens back out of the paged INT4 cache: keys dequantized
// as code * s - zp * s (one multiplication, then one fused multiply-add, in
// float32, rounded once to the output type) and values widened or rounded to
// it, as dense rows [tokens, heads, head_dim].
//
// A page-head slab of the pools is contiguous, a dense row of one head is a
// 128-1024 byte piece, so a warp takes one (sequence, page, head): it loads
// the group's scale / zero-point once, each lane 8 channels of them, and
// streams the slab's 16 rows with 4-byte code loads and 16-byte value loads,
// several rows in flight. Nothing is reused, so it is bound by HBM bytes: 8 x 4096
// tokens of 32 x 128 float32 in 291 to 298 us, 5.7 TB/s; bfloat16 199 us, 4.4 TB/s. A CTA's
// warps are heads, so with few heads most of them have nothing to do: 64 x 4096 bfloat16
// tokens of 8 heads 4.5 TB/s, of 2 heads 3.4, of 1 head 2.7.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "../../include/int4kv_b200.h"

using namespace i4kv;

namespace {

constexpr int kReadWarps = 8;

struct ReadArgs {
  const uint8_t* k_pool;
  const void* v_pool;       // nullable
  const float* sz_pool;
  const int32_t* block_table;
  const int32_t* start;     // [B] first token read
  const int32_t* tok_off;   // [B+1] output rows of each sequence
  int num_rows, max_rows;   // rows of the outputs; bound of one sequence's rows
  int heads, dim, group_tokens, page, max_pages, num_pages;
  void* k_out;
  void* v_out;              // null with v_pool
  uint32_t* status;
};

// N consecutive stored values (kind VK) as float32.
template <int VK, int N>
I4KV_DEVINL void load_values(const void* base, size_t i, float* x) {
  if constexpr (VK == INT4KV_VALUES_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const float4 w = __ldcs(p + j);
      x[4 * j] = w.x; x[4 * j + 1] = w.y; x[4 * j + 2] = w.z; x[4 * j + 3] = w.w;
    }
  } else {
    uint32_t w[N / 2];
    const uint16_t* p = static_cast<const uint16_t*>(base) + i;
    if constexpr (N == 8) {
      const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p));
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
      const uint2 q = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = q.x; w[1] = q.y;
    }
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      if constexpr (VK == INT4KV_VALUES_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        x[2 * j] = f.x; x[2 * j + 1] = f.y;
      } else {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
}

template <int OUT, int N>
I4KV_DEVINL void store_values(void* base, size_t i, const float* x) {
  if constexpr (OUT == INT4KV_VALUES_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j)
      __stcs(p + j, make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]));
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      if constexpr (OUT == INT4KV_VALUES_F16) {
        const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    uint16_t* p = static_cast<uint16_t*>(base) + i;
    if constexpr (N == 8)
      __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    else
      __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
  }
}

// N = channels per lane: 8 where they divide head_dim, else 4.
template <int VK, int OUT, int N>
__global__ void __launch_bounds__(kReadWarps * 32) cache_read_kernel(ReadArgs a) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.z, h = blockIdx.x * kReadWarps + (threadIdx.x >> 5);
  const int off = a.tok_off[b], n = a.tok_off[b + 1] - off, start = a.start[b];
  if (n == 0 || h >= a.heads) return;
  // 64-bit sums: malformed metadata must not wrap into range
  if (n < 0 || n > a.max_rows || off < 0 || (long long)off + n > a.num_rows || start < 0 ||
      (long long)start + n > (long long)a.max_pages * a.page) {
    if (a.status && lane == 0) atomicOr(a.status, kStatusBadLength);
    return;
  }
  const int behind = (int)blockIdx.y * a.page;  // from the first page's first token
  if (behind >= start % a.page + n) return;     // (a sum of both could pass 2^31)
  const int pg = start / a.page + (int)blockIdx.y, p0 = pg * a.page;
  const int t0 = max(start, p0), t1 = start + n - p0 < a.page ? start + n : p0 + a.page;
  const int32_t* row = a.block_table + (size_t)b * a.max_pages;
  const int phys = row[pg], home = row[pg * a.page / a.group_tokens * (a.group_tokens / a.page)];
  const bool ok = phys >= 0 && phys < a.num_pages && home >= 0 && home < a.num_pages;
  if (!ok && a.status && lane == 0) atomicOr(a.status, kStatusBadPage);
  const int D = a.dim, per_row = D / N;
  const size_t slab = ((size_t)(ok ? phys : 0) * a.heads + h) * a.page;
  const float* sz = a.sz_pool + ((size_t)(ok ? home : 0) * a.heads + h) * 2 * D;
  const size_t out_row = (size_t)a.heads * D;

  auto params = [&](int c, float* s, float* z) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(sz + c + j));
      const float4 y = __ldg(reinterpret_cast<const float4*>(sz + D + c + j));
      s[j] = x.x; s[j + 1] = x.y; s[j + 2] = x.z; s[j + 3] = x.w;
      z[j] = -(y.x * x.x); z[j + 1] = -(y.y * x.y); z[j + 2] = -(y.z * x.z); z[j + 3] = -(y.w * x.w);
    }
  };
  auto element = [&](int t, int c, const float* s, const float* z) {
    const size_t at = slab + (t - pg * a.page);
    const size_t to = (size_t)(off + t - start) * out_row + (size_t)h * D + c;
    float k[N], v[N];
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = 0.f;
    if (ok) {
      const uint8_t* src = a.k_pool + at * (D / 2) + c / 2;
      if constexpr (N == 8) w = __ldcs(reinterpret_cast<const unsigned int*>(src));
      else w = __ldcs(reinterpret_cast<const unsigned short*>(src));
      if (a.v_pool) load_values<VK, N>(a.v_pool, at * D + c, v);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) k[j] = ok ? fmaf((float)((w >> (4 * j)) & 15u), s[j], z[j]) : 0.f;
    store_values<OUT, N>(a.k_out, to, k);
    if (a.v_pool) store_values<OUT, N>(a.v_out, to, v);
  };

  float s[N], z[N];
  if (32 % per_row == 0) {  // the lane keeps its channels: parameters loaded once
    const int c = (lane % per_row) * N, step = 32 / per_row;
    params(c, s, z);
#pragma unroll 4
    for (int t = t0 + lane / per_row; t < t1; t += step) element(t, c, s, z);
  } else {
    for (int c = lane * N; c < D; c += 32 * N) {
      params(c, s, z);
#pragma unroll 4
      for (int t = t0; t < t1; ++t) element(t, c, s, z);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int VK, int OUT>
void launch_read(const ReadArgs& a, dim3 grid, cudaStream_t stream) {
  if (a.dim % 8 == 0)
    cache_read_kernel<VK, OUT, 8><<<grid, kReadWarps * 32, 0, stream>>>(a);
  else
    cache_read_kernel<VK, OUT, 4><<<grid, kReadWarps * 32, 0, stream>>>(a);
}

template <int VK>
void launch_read_out(int out_dtype, const ReadArgs& a, dim3 grid, cudaStream_t stream) {
  if (out_dtype == INT4KV_VALUES_F32) launch_read<VK, INT4KV_VALUES_F32>(a, grid, stream);
  else if (out_dtype == INT4KV_VALUES_F16) launch_read<VK, INT4KV_VALUES_F16>(a, grid, stream);
  else launch_read<VK, INT4KV_VALUES_BF16>(a, grid, stream);
}

}  // namespace

extern "C" cudaError_t int4kv_cache_read(const uint8_t* k_pool, const void* v_pool, int value_dtype,
                                         const float* sz_pool, const int32_t* block_table,
                                         const int32_t* start_pos, const int32_t* tok_offsets,
                                         int batch, int num_rows, int max_rows_per_seq,
                                         int num_heads, int head_dim, int group_tokens,
                                         int page_tokens, int max_pages, int num_pages,
                                         int out_dtype, void* k_out, void* v_out, uint32_t* status,
                                         cudaStream_t stream) {
  if (batch <= 0 || batch > 65535 || num_rows < 0 || max_rows_per_seq < 0 || num_heads <= 0 ||
      head_dim <= 0 || head_dim % 4 != 0 || max_pages <= 0 || num_pages <= 0)
    return cudaErrorInvalidValue;
  if (page_tokens <= 0 || group_tokens <= 0 || group_tokens % page_tokens != 0) return cudaErrorInvalidValue;
  // (the kernel's loops step past the last token by less than 1024)
  if ((long long)max_pages * page_tokens > 0x7fffffffll - 1024) return cudaErrorInvalidValue;
  for (int kind : {value_dtype, out_dtype})
    if (kind != INT4KV_VALUES_F32 && kind != INT4KV_VALUES_F16 && kind != INT4KV_VALUES_BF16)
      return cudaErrorInvalidValue;
  if (!k_pool || !sz_pool || !block_table || !start_pos || !tok_offsets) return cudaErrorInvalidValue;
  if (num_rows == 0 || max_rows_per_seq == 0) return cudaSuccess;  // (outputs of no rows may have no address)
  if ((v_pool != nullptr) != (v_out != nullptr)) return cudaErrorInvalidValue;
  if (!k_out || !aligned16(k_pool) || !aligned16(sz_pool) || !aligned16(v_pool) || !aligned16(k_out) ||
      !aligned16(v_out))
    return cudaErrorInvalidValue;
  // a range may start inside a page, but it never has more pages than the table
  const long long pages = ((long long)max_rows_per_seq + 2 * page_tokens - 2) / page_tokens;
  const long long y = pages < max_pages ? pages : max_pages;
  if (y > 65535) return cudaErrorInvalidValue;
  ReadArgs a{k_pool, v_pool, sz_pool, block_table, start_pos, tok_offsets, num_rows, max_rows_per_seq,
             num_heads, head_dim, group_tokens, page_tokens, max_pages, num_pages, k_out, v_out, status};
  dim3 grid((num_heads + kReadWarps - 1) / kReadWarps, (unsigned)y, batch);
  if (value_dtype == INT4KV_VALUES_F32) launch_read_out<INT4KV_VALUES_F32>(out_dtype, a, grid, stream);
  else if (value_dtype == INT4KV_VALUES_F16) launch_read_out<INT4KV_VALUES_F16>(out_dtype, a, grid, stream);
  else launch_read_out<INT4KV_VALUES_BF16>(out_dtype, a, grid, stream);
  return cudaGetLastError();
}
