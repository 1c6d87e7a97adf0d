// Batch metadata from request lengths, on the GPU: block tables, slots,
// positions and work lists of a step, with blocks from a ring of free ones.
//
// One launch.  Every workgroup reads all sequences and forms the running sums
// (token rows, block needs, blocks given back, work items) for itself -- a few
// thousand lengths cost less than a second launch or a wait between
// workgroups would -- then does its share of the token rows and returned
// blocks, finding the sequence of a row by binary search of the sums in LDS; the
// first workgroup writes what there is one of per sequence.  All sums come from
// one scan that takes every request for granted; only where the rows or the free
// blocks do not suffice are they formed again step by step.  Blocks are taken
// from the ring's head and returned at its tail, so no workgroup writes an entry
// that another reads; the ring's state is written by the workgroup that is done
// with it last (a ticket in its third word), and so are the lengths where they take
// the place of the ones that every workgroup reads.
// Bound: the launch and a chain of dependent reads (lengths, then table or ring): 32
// decoding sequences 4.2 us, 16k rows of 8 sequences 5.8; of thousands of sequences the
// scan, and what the first workgroup writes alone: 2094 sequences 9.9 us (5 of them in
// each thread; forming the sums twice took 23), 4000 17, 8000 22.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "batch_sums.hpp"
#include "device.hpp"
#include "redline_amd/rlk.h"
#include "status.hpp"

namespace rlk {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / kWave;
constexpr int kRowsPerGroup = kThreads;

struct TableArgs {
  rlk_block_pool pool;
  rlk_batch_tables t;
  int in_place;  // ctx_len is past_len, or q_len is new_len
};

// Exclusive sums of N values over the workgroup's threads (saturating); the
// totals come back in `total`.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*wave_tot)[5]) {
  static_assert(N <= 5, "room for 5 sums");
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

__device__ __forceinline__ int blocks_of(uint32_t tokens, uint32_t bs) {
  const uint32_t b = tokens / bs;
  return static_cast<int>(b * bs == tokens ? b : b + 1);
}

// What one sequence asks for.
struct Request {
  int past, len, have, need, back;  // tokens cached, new; blocks held, needed, returned
  bool live, ended, fits;           // fits: its table row, and past is sound
};

__device__ __forceinline__ Request request(const rlk_batch_tables& t, int past, int n) {
  Request r;
  r.past = past;
  r.live = n > 0;
  r.ended = n < 0;
  r.len = min(max(n, 0), kSat);
  const uint32_t p = max(past, 0);
  r.have = blocks_of(p, t.block_size);
  const int want = blocks_of(p + r.len, t.block_size);  // p + len is below 2^31 + 2^30
  r.need = static_cast<int>(static_cast<uint32_t>(want) - static_cast<uint32_t>(r.have));
  r.back = r.ended ? min(r.have, t.max_blocks_per_seq) : 0;
  r.fits = r.live && past >= 0 && want >= 0 && want <= t.max_blocks_per_seq;
  return r;
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

// kPer: sequences of a thread, which hold its requests in registers.
template <int kPer>
__global__ __launch_bounds__(kThreads) void build_batch_tables_kernel(TableArgs a) {
  const rlk_batch_tables& t = a.t;
  // The sequences of a thread are lines of memory apart where it has many: arrays per
  // sequence are then read and written through LDS, whole lines at a time (8000 sequences
  // 22 us, without 33; 2094 would take 10.6 instead of 10.0).
  constexpr bool kLines = kPer > 5;
  extern __shared__ int lds[];
  __shared__ int wave_tot[kWaves][5];
  __shared__ int taken_s, last_s;
  const int S = t.num_seqs, tid = threadIdx.x, group = blockIdx.x, groups = gridDim.x;
  // per sequence: first row, first taken block (-1: no rows of it, -2: it has ended),
  // tokens before, first returned block
  int* start_of = lds;
  int* base_of = start_of + S;
  int* past_of = base_of + S;
  int* back_of = past_of + S;
  const int cap = a.pool.capacity, mb = t.max_blocks_per_seq, bs = t.block_size, thr = t.decode_query_threshold;
  // (a state outside the ring is brought inside it: no index leaves the ring)
  const int head0 = a.pool.state[0], count = min(max(a.pool.state[1], 0), cap);
  const int head = head0 >= 0 && head0 < cap ? head0 : 0;

  const int per = (S + kThreads - 1) / kThreads;  // at most kPer
  const int s0 = tid * per, mine = max(min(S - s0, per), 0);
  Request req[kPer];
  if constexpr (kLines) {
    for (int s = tid; s < S; s += kThreads) {
      past_of[s] = t.past_len[s];
      start_of[s] = t.new_len[s];
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const bool on = k < mine;
    req[k] = request(t, on ? (kLines ? past_of : t.past_len)[s0 + k] : 0,
                     on ? (kLines ? start_of : t.new_len)[s0 + k] : 0);
  }
  // rows, blocks needed and returned, decode items, prefill and refused
  // sequences (16 bits each), as if every request that fits were granted
  auto items = [&](const Request& r, bool ok, int& dec, int& seqs) {
    dec = ok && r.len <= thr ? r.len : 0;
    seqs = (ok && r.len > thr ? 1 : 0) + (r.live && !ok ? 1 << 16 : 0);
  };
  int sum[5] = {0, 0, 0, 0, 0}, total[5];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    int dec, seqs;
    items(req[k], req[k].fits, dec, seqs);
    sum[0] = sat_add(sum[0], req[k].len);
    sum[1] = sat_add(sum[1], req[k].fits ? req[k].need : 0);
    sum[2] = sat_add(sum[2], req[k].back);
    sum[3] = sat_add(sum[3], dec);
    sum[4] += seqs;
  }
  block_scan(sum, total, wave_tot);
  const bool ample = total[0] <= t.num_rows && total[1] <= count;  // uniform
  if (!ample) {
    // rows first: who fits them; then the needs in order; then who is granted
    int at = sum[0], need[1] = {0}, need_total[1];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      req[k].fits = req[k].fits && req[k].len <= t.num_rows && at <= t.num_rows - req[k].len;
      need[0] = sat_add(need[0], req[k].fits ? req[k].need : 0);
      at = sat_add(at, req[k].len);
    }
    block_scan(need, need_total, wave_tot);
    sum[1] = need[0];
    int before = need[0], last[2] = {0, 0}, last_total[2];
    if (tid == 0) taken_s = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int n = req[k].fits ? req[k].need : 0;
      const bool ok = req[k].fits && (n == 0 || (before <= count && n <= count - before));
      int dec, seqs;
      items(req[k], ok, dec, seqs);
      last[0] = sat_add(last[0], dec);
      last[1] += seqs;
      // granted needs are a prefix of the needs
      if (ok && n > 0) atomicMax(&taken_s, before + n);
      before = sat_add(before, n);
    }
    block_scan(last, last_total, wave_tot);
    sum[3] = last[0];
    sum[4] = last[1];
    total[1] = taken_s;
    total[3] = last_total[0];
    total[4] = last_total[1];
  }
  const int taken = total[1], pre_total = total[4] & 0xffff;
  {
    int start = sum[0], need = sum[1], back = sum[2], dec = sum[3], pre = sum[4] & 0xffff;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k < mine) {
        const Request& r = req[k];
        const int s = s0 + k, n = r.fits ? r.need : 0;
        const bool ok = r.fits && (n == 0 || (need <= count && n <= count - need));
        start_of[s] = start;
        base_of[s] = ok ? need : (r.ended ? -2 : -1);
        past_of[s] = r.past;
        back_of[s] = back;
        if (group == 0) {
          if (!kLines && !a.in_place) {
            t.q_start[s] = start;
            t.q_len[s] = ok ? r.len : 0;
            t.ctx_len[s] = ok ? r.past + r.len : (r.ended ? 0 : r.past);
          }
          if (ok && r.len <= thr) {
            for (int i = 0; i < r.len; ++i) {
              t.decode_token[dec + i] = start + i;
              t.decode_seq[dec + i] = s;
            }
          }
          if (ok && r.len > thr) t.prefill_seq[pre] = s;
        }
        if (ok && r.len <= thr) dec += r.len;
        if (ok && r.len > thr) pre += 1;
        need = sat_add(need, n);
        back = sat_add(back, r.back);
        start = sat_add(start, r.len);
      }
    }
  }
  if (group == 0) {
    for (int i = total[3] + tid; i < t.num_rows; i += kThreads) {
      t.decode_token[i] = -1;
      t.decode_seq[i] = 0;
    }
    for (int i = pre_total + tid; i < S; i += kThreads) t.prefill_seq[i] = -1;
    if (tid == 0) {
      t.counts[0] = total[0];
      t.counts[1] = total[3];
      t.counts[2] = pre_total;
      t.counts[3] = total[4] >> 16;
    }
  }
  __syncthreads();
  // lengths of the sequences first, first + step, .. from the sums
  auto write_lengths = [&](int first, int step) {
    for (int s = first; s < S; s += step) {
      // (a granted sequence's sums are not saturated)
      const int start = start_of[s], len = (s + 1 < S ? start_of[s + 1] : total[0]) - start;
      const int base = base_of[s];
      t.q_start[s] = start;
      t.q_len[s] = base >= 0 ? len : 0;
      t.ctx_len[s] = base >= 0 ? past_of[s] + len : (base == -2 ? 0 : past_of[s]);
    }
  };
  if (kLines && !a.in_place) write_lengths(group * kThreads + tid, groups * kThreads);

  auto ring_at = [&](int i) {  // entry i from the head
    const uint32_t x = static_cast<uint32_t>(head) + static_cast<uint32_t>(i);  // i <= cap
    return static_cast<int>(x >= static_cast<uint32_t>(cap) ? x - cap : x);
  };
  const int row = group * kRowsPerGroup + tid;
  if (row < t.num_rows) {
    int pos = 0, slot = -1;
    if (row < total[0]) {
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
  const int returned = min(total[2], cap - count);
  for (int i = group * kThreads + tid; i < returned; i += groups * kThreads) {
    const int s = find(back_of, S, i);
    a.pool.ring[ring_at(count + i)] = t.block_tables[static_cast<int64_t>(s) * mb + (i - back_of[s])];
  }
  if (tid == 0) {
    int32_t* state = a.pool.state;
    int32_t* out = a.pool.state_out != nullptr ? a.pool.state_out : state;
    // with several workgroups the one whose ticket is the last: every other has
    // read the state, and the lengths
    const bool last = groups == 1 || atomicAdd(&state[2], 1) == groups - 1;
    last_s = last;
    if (last) {
      if (groups > 1) state[2] = 0;
      out[0] = ring_at(taken);
      out[1] = count - taken + returned;
    }
  }
  if (a.in_place) {
    __syncthreads();
    if (last_s) write_lengths(tid, kThreads);
  }
}

template <int kPer>
int launch_tables(const TableArgs& a, hipStream_t stream) {
  const char* what = "build_batch_tables";
  const size_t lds = static_cast<size_t>(a.t.num_seqs) * 4 * sizeof(int);
  if (lds > 48 * 1024) {
    const hipError_t e = grant_dynamic_lds(reinterpret_cast<const void*>(build_batch_tables_kernel<kPer>),
                                           RLK_BATCH_TABLES_MAX_SEQS * 4 * sizeof(int));
    if (e != hipSuccess) return fail(static_cast<int>(e), "%s: %s", what, hipGetErrorString(e));
  }
  const int groups = std::max(1, (a.t.num_rows + kRowsPerGroup - 1) / kRowsPerGroup);
  build_batch_tables_kernel<kPer><<<groups, kThreads, lds, stream>>>(a);
  return launch_status(what);
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
  // every workgroup reads past_len and new_len: what is written must not lie there, but
  // for the lengths themselves (`same`), which are then written last
  struct Out {
    const int32_t* at;
    int64_t n;
    const int32_t* same;
  };
  const int64_t S = t.num_seqs, rows = t.num_rows;
  for (const int32_t* in : {t.past_len, t.new_len})
    for (const Out& o : {Out{t.q_len, S, t.new_len}, Out{t.ctx_len, S, t.past_len}, Out{t.q_start, S, nullptr},
                         Out{t.prefill_seq, S, nullptr}, Out{t.block_tables, S * t.max_blocks_per_seq, nullptr},
                         Out{t.positions, rows, nullptr}, Out{t.slot_mapping, rows, nullptr},
                         Out{t.decode_token, rows, nullptr}, Out{t.decode_seq, rows, nullptr},
                         Out{t.counts, 4, nullptr}})
      if (S > 0 && o.n > 0 && in < o.at + o.n && o.at < in + S && !(in == o.same && o.at == o.same))
        return fail(RLK_EINVAL, "%s: past_len and new_len must not overlap what is written (ctx_len may be "
                                "past_len, q_len new_len)", what);
  const TableArgs a = {*pool, t, t.num_seqs > 0 && (t.ctx_len == t.past_len || t.q_len == t.new_len)};
  // (2560 sequences: 5 a thread 10.3 us, the form for up to 16, which spills scalar
  // registers, 15.1; 2561 take 15.5 by it)
  const int per = (t.num_seqs + kThreads - 1) / kThreads;
  if (per <= 1) return launch_tables<1>(a, stream);
  if (per <= 5) return launch_tables<5>(a, stream);
  static_assert(RLK_BATCH_TABLES_MAX_SEQS <= 16 * kThreads, "16 sequences a thread at most");
  return launch_tables<16>(a, stream);
}
