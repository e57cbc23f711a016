// The note a run leaves of its last stream where that goes on in later runs, and what
// the merge asks of it before it takes addresses from it.
#pragma once

#ifdef __CUDACC__
#define I4KV_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define I4KV_HOST_DEVICE inline
#endif

namespace i4kv {

// The stream at the end of a run that began in it and goes on in later runs, up to
// run `last` (rows 0: there is none): what the merge has to know.
struct RunTail {
  int rows, row0, head, first_row;  // rows of the sequence, its first row; the chunk's
  int slot, last;                   // this run's record of it; the last run that shares it
  int pad[2];
};

// Whether run `run` of `runs` may have left note `n`: every row of outputs [total_rows,
// kv_heads, group_q], record and run that it names is there. Each run writes an empty
// note before it waits for anything, so that a run that fails leaves none; this
// is the second bar, for a note that nobody wrote at all (the workspace is not cleared).
I4KV_HOST_DEVICE bool tail_in_range(const RunTail& n, int run, int runs, int total_rows, int kv_heads, int group_q) {
  if (n.rows <= 0 || n.row0 < 0 || n.head < 0 || n.head >= kv_heads || n.first_row < 0 || n.first_row >= n.rows)
    return false;
  if ((long long)n.row0 * group_q + n.rows > (long long)total_rows * group_q) return false;
  return (n.slot == 2 * run || n.slot == 2 * run + 1) && n.last > run && n.last < runs;
}

}  // namespace i4kv
