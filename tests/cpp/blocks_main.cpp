// Host-only check of the C++ launchers of the block-scaled cache and the batch
// tables: argument errors throw redline::Error before anything is launched;
// empty calls are no-ops.
#include <cstdio>
#include <string>

#include "redline_amd/kernels.h"

using namespace redline;

static int failures = 0;

template <typename F>
static void expect_throw(const char* what, F f, const char* needle) {
  try {
    f();
    std::printf("FAIL %s: no exception\n", what);
    ++failures;
  } catch (const Error& e) {
    if (std::string(e.what()).find(needle) == std::string::npos) {
      std::printf("FAIL %s: message '%s'\n", what, e.what());
      ++failures;
    }
  }
}

int main() {
  alignas(16) static unsigned char dummy[256];
  half* h = reinterpret_cast<half*>(dummy);
  int32_t* i = reinterpret_cast<int32_t*>(dummy);
  float* f = reinterpret_cast<float*>(dummy);
  kernels::KVBlockView kv{dummy, dummy, f, f, 4, 16, 2, 80, static_cast<int>(kernels::KVBlockFormat::kFP8)};
  kernels::BlockAttentionParams p{reinterpret_cast<const uint16_t*>(h), 512, reinterpret_cast<uint16_t*>(h),
                                  4, 0.1f, kv, i, 2, i};
  kernels::DecodeAttentionWork dw;
  dw.num_items = 1;
  kernels::PrefillAttentionWork pw;
  pw.num_seqs = pw.max_q_tiles = 1;
  expect_throw("write", [&] { kernels::rope_and_write_kv_blocks(h, i, i, 1, 4, f, f, kv, nullptr, nullptr); },
               "unsupported head_dim 80");
  expect_throw("read", [&] { kernels::read_kv_blocks(kv, i, 1, h, h, nullptr); }, "unsupported head_dim 80");
  expect_throw("decode", [&] { kernels::paged_attention_decode_blocks(p, dw, nullptr); }, "unsupported head_dim 80");
  expect_throw("prefill", [&] { kernels::paged_attention_prefill_blocks(p, pw, nullptr); },
               "unsupported head_dim 80");
  kernels::BlockPool pool{i, 0, i, nullptr};
  kernels::BatchTables t{};
  t.num_seqs = t.num_rows = 1;
  t.block_size = 16;
  t.max_blocks_per_seq = 1;
  expect_throw("tables", [&] { kernels::build_batch_tables(pool, t, nullptr); }, "ring capacity 0");
  t.num_seqs = t.num_rows = 0;
  dw.num_items = pw.num_seqs = 0;
  try {
    kernels::rope_and_write_kv_blocks(nullptr, nullptr, nullptr, 0, 4, nullptr, nullptr, kv, nullptr, nullptr);
    kernels::read_kv_blocks(kv, nullptr, 0, nullptr, nullptr, nullptr);
    kernels::paged_attention_decode_blocks(p, dw, nullptr);
    kernels::paged_attention_prefill_blocks(p, pw, nullptr);
    kernels::build_batch_tables(pool, t, nullptr);
  } catch (const Error& e) {
    std::printf("FAIL empty call: %s\n", e.what());
    ++failures;
  }
  if (failures == 0) std::printf("PASS\n");
  return failures;
}
