// Batch metadata from request lengths, on the GPU: block tables, slots,
// positions and work lists of a step, with blocks from a ring of free ones.
//
// One launch.  Every workgroup reads all sequences and forms the running sums
// (token rows, block needs, blocks given back, work items) for itself -- a few
// thousand lengths cost less than a second launch or a wait between
// workgroups would -- then does its share of the sequences, token rows and
// returned blocks, finding the sequence of a row by binary search of the sums
// in LDS.  Blocks are taken from the ring's head and returned at its tail, so
// no workgroup writes an entry that another reads; the ring's state is written
// by the workgroup that finishes reading it last (a ticket in its third word).
// Bound: the launch and a chain of two dependent reads (lengths, table or ring).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "device.hpp"
#include "redline_amd/rlk.h"
#include "status.hpp"

namespace rlk {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / kWave;
constexpr int kRowsPerGroup = 2048;
constexpr int kSat = 1 << 30;  // running sums of rows saturate here

struct TableArgs {
  rlk_block_pool pool;
  rlk_batch_tables t;
};

__device__ __forceinline__ int sat_add(int a, int b) { return min(a + b, kSat); }  // a, b <= kSat

// Exclusive sums of N values over the workgroup's threads (saturating); the
// totals come back in `total`.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*wave_tot)[N]) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int incl[N];
#pragma unroll
  for (int k = 0; k < N; ++k) incl[k] = v[k];
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int u = __shfl_up(incl[k], o, kWave);
      if (lane >= o) incl[k] = sat_add(incl[k], u);
    }
  }
  __syncthreads();  // wave_tot of an earlier scan has been read
  if (lane == kWave - 1) {
#pragma unroll
    for (int k = 0; k < N; ++k) wave_tot[wave][k] = incl[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before = sat_add(before, wave_tot[w][k]);
      all = sat_add(all, wave_tot[w][k]);
    }
    // exclusive sum of this thread: the sums of the lanes and waves before it
    const int up = __shfl_up(incl[k], 1, kWave);
    v[k] = sat_add(before, lane > 0 ? up : 0);
    total[k] = all;
  }
}

// What one sequence asks for.
struct Request {
  int past, len, have, want;
  bool live, ended;
};

__device__ __forceinline__ int blocks_of(uint32_t tokens, uint32_t bs) {
  const uint32_t b = tokens / bs;
  return static_cast<int>(b * bs == tokens ? b : b + 1);
}

__device__ __forceinline__ Request request(const rlk_batch_tables& t, int s) {
  Request r;
  const int n = t.new_len[s];
  r.past = t.past_len[s];
  r.live = n > 0;
  r.ended = n < 0;
  r.len = min(max(n, 0), kSat);
  const uint32_t past = max(r.past, 0);
  r.have = blocks_of(past, t.block_size);
  r.want = blocks_of(past + r.len, t.block_size);  // below 2^31 + 2^30
  return r;
}

// Whether a live sequence fits its table row and the token rows.
__device__ __forceinline__ bool fits(const rlk_batch_tables& t, const Request& r, int start) {
  return r.live && r.past >= 0 && r.want >= 0 && r.want <= t.max_blocks_per_seq && r.len <= t.num_rows &&
         start <= t.num_rows - r.len;
}

// Last s in [0, n) with at[s] <= x (at[0] == 0 <= x).
__device__ __forceinline__ int find(const int* at, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (at[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void build_batch_tables_kernel(TableArgs a) {
  const rlk_batch_tables& t = a.t;
  extern __shared__ int lds[];
  __shared__ int wave_tot[kWaves][3];
  const int S = t.num_seqs, tid = threadIdx.x, group = blockIdx.x, groups = gridDim.x;
  // per sequence: first row, first taken block (-1: no rows of it), tokens
  // before, first returned block
  int* start_of = lds;
  int* base_of = start_of + S;
  int* past_of = base_of + S;
  int* back_of = past_of + S;
  const int cap = a.pool.capacity, mb = t.max_blocks_per_seq, bs = t.block_size;
  // (a state outside the ring is brought inside it: no index leaves the ring)
  const int head0 = a.pool.state[0], count = min(max(a.pool.state[1], 0), cap);
  const int head = head0 >= 0 && head0 < cap ? head0 : 0;

  const int per = (S + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, S), s1 = min(s0 + per, S);
  int rows[1] = {0}, rows_total[1];
  for (int s = s0; s < s1; ++s) rows[0] = sat_add(rows[0], request(t, s).len);
  block_scan(rows, rows_total, reinterpret_cast<int(*)[1]>(wave_tot));

  int blk[2] = {0, 0}, blk_total[2];  // needed, returned
  int start = rows[0];
  for (int s = s0; s < s1; ++s) {
    const Request r = request(t, s);
    if (fits(t, r, start)) blk[0] = sat_add(blk[0], r.want - r.have);
    if (r.ended) blk[1] = sat_add(blk[1], min(r.have, mb));
    start = sat_add(start, r.len);
  }
  block_scan(blk, blk_total, reinterpret_cast<int(*)[2]>(wave_tot));

  // decode items, prefill sequences, refused sequences; and the blocks taken
  // (granted needs are a prefix of the needs)
  int item[3] = {0, 0, 0}, item_total[3];
  start = rows[0];
  int need = blk[0];
  auto granted = [&](const Request& r, int at, int before) {
    const int n = r.want - r.have;
    return fits(t, r, at) && (n == 0 || (before <= count && n <= count - before));
  };
  for (int s = s0; s < s1; ++s) {
    const Request r = request(t, s);
    const bool ok = granted(r, start, need);
    if (ok && r.len <= t.decode_query_threshold) item[0] = sat_add(item[0], r.len);
    if (ok && r.len > t.decode_query_threshold) item[1] += 1;
    if (r.live && !ok) item[2] += 1;
    if (fits(t, r, start)) need = sat_add(need, r.want - r.have);
    start = sat_add(start, r.len);
  }
  block_scan(item, item_total, wave_tot);

  start = rows[0];
  need = blk[0];
  int back = blk[1], dec = item[0], pre = item[1];
  for (int s = s0; s < s1; ++s) {
    const Request r = request(t, s);
    const bool ok = granted(r, start, need);
    start_of[s] = start;
    base_of[s] = ok ? need : -1;
    past_of[s] = r.past;
    back_of[s] = back;
    if (group == 0) {
      t.q_start[s] = start;
      t.q_len[s] = ok ? r.len : 0;
      t.ctx_len[s] = ok ? r.past + r.len : (r.ended ? 0 : r.past);
      if (ok && r.len <= t.decode_query_threshold) {
        for (int i = 0; i < r.len; ++i) {
          t.decode_token[dec + i] = start + i;
          t.decode_seq[dec + i] = s;
        }
      }
      if (ok && r.len > t.decode_query_threshold) t.prefill_seq[pre] = s;
    }
    if (ok && r.len <= t.decode_query_threshold) dec += r.len;
    if (ok && r.len > t.decode_query_threshold) pre += 1;
    if (fits(t, r, start)) need = sat_add(need, r.want - r.have);
    if (r.ended) back = sat_add(back, min(r.have, mb));
    start = sat_add(start, r.len);
  }
  if (group == 0) {
    for (int i = item_total[0] + tid; i < t.num_rows; i += kThreads) {
      t.decode_token[i] = -1;
      t.decode_seq[i] = 0;
    }
    for (int i = item_total[1] + tid; i < S; i += kThreads) t.prefill_seq[i] = -1;
    if (tid == 0) {
      t.counts[0] = rows_total[0];
      t.counts[1] = item_total[0];
      t.counts[2] = item_total[1];
      t.counts[3] = item_total[2];
    }
  }
  __syncthreads();

  auto ring_at = [&](int i) {  // entry i from the head
    const uint32_t x = static_cast<uint32_t>(head) + static_cast<uint32_t>(i);  // i <= cap
    return static_cast<int>(x >= static_cast<uint32_t>(cap) ? x - cap : x);
  };
  const int r_end = min((group + 1) * kRowsPerGroup, t.num_rows);
  for (int row = group * kRowsPerGroup + tid; row < r_end; row += kThreads) {
    int pos = 0, slot = -1;
    if (row < rows_total[0]) {
      const int s = find(start_of, S, row);
      if (base_of[s] >= 0) {
        const int past = past_of[s], have = blocks_of(past, bs);
        pos = past + (row - start_of[s]);
        const int b = pos / bs, off = pos - b * bs;
        int32_t* entry = t.block_tables + static_cast<int64_t>(s) * mb + b;
        int id;
        if (b >= have) {  // a block of this step: its first token enters it
          id = a.pool.ring[ring_at(base_of[s] + b - have)];
          if (off == 0) *entry = id;
        } else {
          id = *entry;
        }
        slot = id * bs + off;
      }
    }
    t.positions[row] = pos;
    t.slot_mapping[row] = slot;
  }
  // blocks of ended sequences, behind the free ones
  const int returned = min(blk_total[1], cap - count);
  for (int i = group * kThreads + tid; i < returned; i += groups * kThreads) {
    const int s = find(back_of, S, i);
    a.pool.ring[ring_at(count + i)] = t.block_tables[static_cast<int64_t>(s) * mb + (i - back_of[s])];
  }

  // Taken: needs are granted in order until one exceeds the count, so the sum
  // is the largest prefix of whole requests within it.
  __shared__ int taken_s;
  if (tid == 0) taken_s = 0;
  __syncthreads();
  if (blk_total[0] <= count) {
    if (tid == 0) taken_s = blk_total[0];
  } else {
    for (int s = s0; s < s1; ++s)
      if (base_of[s] >= 0) {
        const Request r = request(t, s);
        if (r.want > r.have) atomicMax(&taken_s, base_of[s] + r.want - r.have);
      }
  }
  __syncthreads();
  if (tid == 0) {
    int32_t* state = a.pool.state;
    int32_t* out = a.pool.state_out != nullptr ? a.pool.state_out : state;
    const int taken = taken_s;
    const int left = count - taken + returned;
    if (groups == 1) {
      out[0] = ring_at(taken);
      out[1] = left;
    } else if (atomicAdd(&state[2], 1) == groups - 1) {  // every group has read the state
      state[2] = 0;
      out[0] = ring_at(taken);
      out[1] = left;
    }
  }
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_build_batch_tables(const rlk_block_pool* pool, const rlk_batch_tables* tables,
                                      hipStream_t stream) {
  const char* what = "build_batch_tables";
  if (pool == nullptr || tables == nullptr) return fail(RLK_EINVAL, "%s: null pool or tables", what);
  const rlk_batch_tables& t = *tables;
  if (t.num_seqs < 0 || t.num_rows < 0 || t.num_rows > kSat)
    return fail(RLK_EINVAL, "%s: bad sequence count %d or row count %d", what, t.num_seqs, t.num_rows);
  if (t.num_seqs == 0 && t.num_rows == 0) return RLK_OK;
  if (t.num_seqs > RLK_BATCH_TABLES_MAX_SEQS)
    return fail(RLK_EUNSUPPORTED, "%s: %d sequences exceed %d; split the batch", what, t.num_seqs,
                RLK_BATCH_TABLES_MAX_SEQS);
  if (t.block_size <= 0 || t.max_blocks_per_seq <= 0 || t.decode_query_threshold < 0 ||
      pool->capacity <= 0 || pool->capacity > kSat)
    return fail(RLK_EINVAL, "%s: bad block size %d, table width %d, decode threshold %d or ring "
                            "capacity %d", what, t.block_size, t.max_blocks_per_seq,
                t.decode_query_threshold, pool->capacity);
  if (static_cast<int64_t>(t.block_size) * t.max_blocks_per_seq > 0x7fffffffll)
    return fail(RLK_EINVAL, "%s: table rows of %d blocks of %d exceed 32-bit positions", what,
                t.max_blocks_per_seq, t.block_size);
  if (pool->ring == nullptr || pool->state == nullptr || t.counts == nullptr ||
      (t.num_seqs > 0 && (t.past_len == nullptr || t.new_len == nullptr || t.block_tables == nullptr ||
                          t.q_start == nullptr || t.q_len == nullptr || t.ctx_len == nullptr ||
                          t.prefill_seq == nullptr)) ||
      (t.num_rows > 0 && (t.positions == nullptr || t.slot_mapping == nullptr ||
                          t.decode_token == nullptr || t.decode_seq == nullptr)))
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  const size_t lds = static_cast<size_t>(t.num_seqs) * 4 * sizeof(int);
  if (lds > 48 * 1024) {
    const hipError_t e = grant_dynamic_lds(reinterpret_cast<const void*>(build_batch_tables_kernel),
                                           RLK_BATCH_TABLES_MAX_SEQS * 4 * sizeof(int));
    if (e != hipSuccess)
      return fail(static_cast<int>(e), "%s: %s", what, hipGetErrorString(e));
  }
  const int groups = std::max(1, (t.num_rows + kRowsPerGroup - 1) / kRowsPerGroup);
  const TableArgs a = {*pool, t};
  build_batch_tables_kernel<<<groups, kThreads, lds, stream>>>(a);
  return launch_status(what);
}
