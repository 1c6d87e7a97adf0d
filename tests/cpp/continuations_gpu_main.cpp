// GPU test of the C++ header's extensions for many continuations of one prompt: a
// prompt and a token of each continuation are normed, rotated and written to a paged
// cache (rope_and_write_kv_norm), read back (read_kv), attended to with the prompt
// shared (paged_attention_decode_shared), and tokens drawn (sample_tokens); each against
// the formulas in 64 bits.
//
// Prints one line per check and PASS or FAIL at the end; exit status 0 only on PASS.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <exception>
#include <numeric>
#include <vector>

#include "redline_amd/kernels.h"

using namespace redline;

namespace {

int failures = 0;

#define HIP_OK(x)                                                                    \
  do {                                                                               \
    const hipError_t e_ = (x);                                                       \
    if (e_ != hipSuccess) {                                                          \
      std::printf("HIP error %s at %s:%d\n", hipGetErrorString(e_), __FILE__, __LINE__); \
      std::exit(2);                                                                  \
    }                                                                                \
  } while (0)

template <typename To, typename T>
To* upload(const std::vector<T>& h) {
  void* d = nullptr;
  HIP_OK(hipMalloc(&d, h.size() * sizeof(T)));
  HIP_OK(hipMemcpy(d, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice));
  return static_cast<To*>(d);
}
template <typename T>
std::vector<T> download(const void* d, size_t n) {
  std::vector<T> h(n);
  HIP_OK(hipMemcpy(h.data(), d, n * sizeof(T), hipMemcpyDeviceToHost));
  return h;
}
void report(const char* what, bool ok, double worst) {
  std::printf("%s %s (worst share of the bound %.3g)\n", ok ? "ok  " : "FAIL", what, worst);
  failures += !ok;
}

uint32_t state = 12345;
float uniform() {  // (0, 1)
  state = state * 1664525u + 1013904223u;
  return (static_cast<float>(state >> 8) + 0.5f) * 0x1p-24f;
}

}  // namespace

int main() {
  constexpr int kPrompt = 300, kItems = 3, T = kPrompt + kItems, Hq = 4, Hkv = 2, D = 64, BS = 16;
  constexpr int kPromptBlocks = (kPrompt + BS - 1) / BS, MB = kPromptBlocks + 1, kCols = (Hq + 2 * Hkv) * D;
  constexpr double u16 = 0x1p-11, u32 = 0x1p-24;
  hipStream_t stream;
  HIP_OK(hipStreamCreate(&stream));

  // The prompt's whole blocks are shared; each continuation has a block of its own for the rest of
  // the prompt and its token.
  constexpr int kShared = kPrompt / BS * BS;
  const int blocks = kPromptBlocks + kItems;
  std::vector<_Float16> qkv(T * kCols), qn(D), kn(D);
  for (auto& x : qkv) x = static_cast<_Float16>(4.f * uniform() - 2.f);
  for (int i = 0; i < D; ++i) {
    qn[i] = static_cast<_Float16>(0.5f + uniform());
    kn[i] = static_cast<_Float16>(0.5f + uniform());
  }
  std::vector<int32_t> pos(T), slots(T), table(kItems * MB), items(kItems), seqs(kItems);
  for (int t = 0; t < kPrompt; ++t) pos[t] = slots[t] = t;
  for (int i = 0; i < kItems; ++i) {
    pos[kPrompt + i] = kPrompt;
    slots[kPrompt + i] = (kPromptBlocks + i) * BS + kPrompt % BS;
    for (int b = 0; b < MB; ++b) table[i * MB + b] = b < kShared / BS ? b : (b == kShared / BS ? kPromptBlocks + i : 0);
    items[i] = kPrompt + i;
    seqs[i] = i;
  }
  std::vector<float> cos(static_cast<size_t>(kPrompt + 1) * D / 2), sin(cos.size());
  for (int p = 0; p <= kPrompt; ++p)
    for (int i = 0; i < D / 2; ++i) {
      const double angle = p * std::pow(10000.0, -2.0 * i / D);
      cos[p * (D / 2) + i] = static_cast<float>(std::cos(angle));
      sin[p * (D / 2) + i] = static_cast<float>(std::sin(angle));
    }
  const size_t cells = static_cast<size_t>(blocks) * Hkv * BS * D;
  KVLayerView kv;
  kv.k = upload<half>(std::vector<_Float16>(cells, static_cast<_Float16>(0.f)));
  kv.v = upload<half>(std::vector<_Float16>(cells, static_cast<_Float16>(0.f)));
  kv.block_size = BS;
  kv.num_kv_heads = Hkv;
  kv.head_dim = D;
  kv.dtype = KVDType::kFP16;
  half* d_qkv = upload<half>(qkv);
  int32_t *d_pos = upload<int32_t>(pos), *d_slots = upload<int32_t>(slots);

  kernels::NormRopeOptions opt = {};
  opt.q_norm = upload<uint16_t>(qn);
  opt.k_norm = upload<uint16_t>(kn);
  opt.eps = 1e-6f;
  kernels::rope_and_write_kv_norm(d_qkv, d_pos, d_slots, T, Hq, upload<float>(cos), upload<float>(sin), kv, opt, stream);
  half* d_k = upload<half>(std::vector<_Float16>(T * Hkv * D));
  half* d_v = upload<half>(std::vector<_Float16>(T * Hkv * D));
  kernels::read_kv(kv, d_slots, T, d_k, d_v, RLK_SCALE_F32, stream);
  HIP_OK(hipStreamSynchronize(stream));
  const auto q_out = download<_Float16>(d_qkv, qkv.size());
  const auto k_out = download<_Float16>(d_k, T * Hkv * D), v_out = download<_Float16>(d_v, T * Hkv * D);
  {
    double worst = 0;
    bool same_v = true;
    for (int t = 0; t < T; ++t)
      for (int h = 0; h < Hq + Hkv; ++h) {
        const _Float16* x = &qkv[t * kCols + h * D];
        const _Float16* y = h < Hq ? &q_out[t * kCols + h * D] : &k_out[(t * Hkv + h - Hq) * D];
        const auto& w = h < Hq ? qn : kn;
        double sum = 0;
        for (int i = 0; i < D; ++i) sum += static_cast<double>(x[i]) * x[i];
        const double r = 1.0 / std::sqrt(sum / D + opt.eps);
        for (int i = 0; i < D / 2; ++i) {
          const double a = x[i] * r * w[i], b = x[i + D / 2] * r * w[i + D / 2];
          const double c = cos[pos[t] * (D / 2) + i], s = sin[pos[t] * (D / 2) + i];
          // one rounding to fp16; in fp32 a sum of D squares, root, and five products and sums
          const double lo = a * c - b * s, hi = b * c + a * s, room = (D + 16) * u32 * (std::fabs(a) + std::fabs(b)) + 0x1p-25;
          worst = std::max(worst, std::fabs(y[i] - lo) / (u16 * std::fabs(lo) + room));
          worst = std::max(worst, std::fabs(y[i + D / 2] - hi) / (u16 * std::fabs(hi) + room));
        }
      }
    for (int t = 0; t < T; ++t)
      same_v = same_v && std::memcmp(&v_out[t * Hkv * D], &qkv[t * kCols + (Hq + Hkv) * D], Hkv * D * 2) == 0;
    report("rope_and_write_kv_norm, read_kv", worst <= 1.0 && same_v, worst);
  }

  {
    half* kp = static_cast<half*>(kv.k);
    half* vp = static_cast<half*>(kv.v);
    for (int i = 0; i < kItems; ++i)
      for (int h = 0; h < Hkv; ++h) {
        const size_t rows = static_cast<size_t>(kPrompt - kShared) * D;
        const size_t src = (static_cast<size_t>(kShared / BS) * Hkv + h) * BS * D;
        const size_t dst = (static_cast<size_t>(kPromptBlocks + i) * Hkv + h) * BS * D;
        HIP_OK(hipMemcpy(kp + dst, kp + src, rows * 2, hipMemcpyDeviceToDevice));
        HIP_OK(hipMemcpy(vp + dst, vp + src, rows * 2, hipMemcpyDeviceToDevice));
      }
    kernels::AttentionParams p;
    half* out = upload<half>(std::vector<_Float16>(T * Hq * D));
    p.q = d_qkv;
    p.q_stride = kCols;
    p.out = out;
    p.num_heads = Hq;
    p.scale = 0.125f;
    p.kv = kv;
    p.block_tables = upload<int32_t>(table);
    p.max_blocks_per_seq = MB;
    p.positions = d_pos;
    kernels::SharedPrefixWork w = {};
    w.item_token = upload<int32_t>(items);
    w.item_seq = upload<int32_t>(seqs);
    w.num_items = kItems;
    w.group_start = upload<int32_t>(std::vector<int32_t>{0, kItems});
    w.group_prefix = upload<int32_t>(std::vector<int32_t>{kShared});
    w.num_groups = 1;
    w.max_group_items = kItems;
    w.max_prefix_partitions = (kShared + 255) / 256;
    w.max_partitions = 1;
    const size_t parts = static_cast<size_t>(kItems) * Hq * (w.max_prefix_partitions + 1);
    w.ws_out = upload<float>(std::vector<float>(parts * D));
    w.ws_max = upload<float>(std::vector<float>(parts));
    w.ws_sum = upload<float>(std::vector<float>(parts));
    kernels::paged_attention_decode_shared(p, w, RLK_SCALE_F32, stream);
    HIP_OK(hipStreamSynchronize(stream));
    const auto o = download<_Float16>(out, T * Hq * D);
    double worst = 0;
    for (int i = 0; i < kItems; ++i)
      for (int h = 0; h < Hq; ++h) {
        const int t = kPrompt + i, g = h / (Hq / Hkv), n = kPrompt + 1;
        std::vector<double> s(n), num(D), size(D), big(D);
        auto row = [&](int key) { return (static_cast<size_t>(key < kPrompt ? key : t) * Hkv + g) * D; };
        double most = -1e300, amp = 0, sum = 0;
        for (int key = 0; key < n; ++key) {
          double dot = 0, abs = 0;
          for (int d = 0; d < D; ++d) {
            const double x = static_cast<double>(q_out[t * kCols + h * D + d]) * k_out[row(key) + d];
            dot += x;
            abs += std::fabs(x);
          }
          s[key] = dot * p.scale;
          amp = std::max(amp, abs * p.scale);
          most = std::max(most, s[key]);
        }
        for (int key = 0; key < n; ++key) {
          const double e = std::exp(s[key] - most);
          sum += e;
          for (int d = 0; d < D; ++d) {
            const double v = v_out[row(key) + d];
            num[d] += e * v;
            size[d] += e * std::fabs(v);
            big[d] = std::max(big[d], std::fabs(v));
          }
        }
        // a score is off by D products and sums and three roundings, a probability by twice that
        // and half a step of fp16 (or 2^-25 of the largest), the sums of n by n roundings
        const double rel = u16 + 3 * (D + 4) * u32 * amp + 2 * n * u32 + 0x1p-20;
        for (int d = 0; d < D; ++d) {
          const double want = num[d] / sum, room = rel * size[d] / sum + n * 0x1p-25 * big[d];
          const double err = std::fabs(o[(t * Hq + h) * D + d] - want);
          worst = std::max(worst, err / (room + u16 * (std::fabs(want) + room) + 0x1p-25));
        }
      }
    report("paged_attention_decode_shared", worst <= 1.0, worst);
    p.scale = NAN;
    bool threw = false;
    try {
      kernels::paged_attention_decode_shared(p, w, RLK_SCALE_F32, stream);
    } catch (const std::exception& e) {
      threw = std::strstr(e.what(), "finite") != nullptr;
    }
    report("paged_attention_decode_shared refuses a scale of NaN", threw, 0);
  }

  {  // tokens of 9000 by the order of the logits
    constexpr int R = 24, V = 9000;
    std::vector<float> x(R * V), temp(R), top_p(R), min_p(R), u(R);
    std::vector<int32_t> top_k(R);
    for (auto& l : x) l = 12.f * uniform();
    for (int r = 0; r < R; ++r) {
      temp[r] = 0.3f + uniform();
      top_k[r] = r % 3 == 0 ? 0 : static_cast<int>(500 * uniform()) + 1;
      top_p[r] = r % 2 == 0 ? 1.f : uniform();
      min_p[r] = r % 4 < 3 ? 0.f : 0.3f * uniform();
      u[r] = uniform();
    }
    kernels::SamplingWork w = {};
    w.logits = upload<float>(x);
    w.logits_fp32 = 1;
    w.row_stride = V;
    w.num_rows = R;
    w.vocab = V;
    w.temperature = upload<float>(temp);
    w.top_k = upload<int32_t>(top_k);
    w.top_p = upload<float>(top_p);
    w.min_p = upload<float>(min_p);
    w.uniform = upload<float>(u);
    w.tokens = upload<int32_t>(std::vector<int32_t>(R, -1));
    w.logprobs = upload<float>(std::vector<float>(R));
    w.workspace_bytes = kernels::sampling_workspace_bytes(R, V);
    w.workspace = upload<char>(std::vector<char>(w.workspace_bytes));
    kernels::sample_tokens(w, stream);
    HIP_OK(hipStreamSynchronize(stream));
    const auto tok = download<int32_t>(w.tokens, R);
    const auto lp = download<float>(w.logprobs, R);
    double worst = 0;
    bool same = true;
    for (int r = 0; r < R; ++r) {
      const float* l = &x[r * V];
      std::vector<int> at(V);
      std::iota(at.begin(), at.end(), 0);
      std::stable_sort(at.begin(), at.end(), [&](int a, int b) { return l[a] > l[b]; });
      std::vector<double> run(V), wt(V);
      for (int j = 0; j < V; ++j) {
        wt[j] = std::exp((static_cast<double>(l[at[j]]) - l[at[0]]) / temp[r]);
        run[j] = wt[j] + (j > 0 ? run[j - 1] : 0);
      }
      int n = top_k[r] > 0 ? std::min(top_k[r], V) : V;
      if (top_p[r] < 1.f) {
        const double target = static_cast<double>(top_p[r]) * run[n - 1];
        int m = 1;
        while (m < n && run[m - 1] < target) ++m;
        n = m;
      }
      while (n > 1 && wt[n - 1] < min_p[r]) --n;
      int j = 0;
      while (j < n - 1 && run[j] <= u[r] * run[n - 1]) ++j;
      const double want = std::log(wt[j] / run[n - 1]);
      if (tok[r] != at[j]) std::printf("row %d: token %d, expected %d\n", r, tok[r], at[j]);
      same = same && tok[r] == at[j];
      worst = std::max(worst, std::fabs(lp[r] - want) / (u32 * std::fabs(want) + 0x1p-32));
    }
    report("sample_tokens", same && worst <= 1.0, worst);
  }

  HIP_OK(hipStreamDestroy(stream));
  std::printf("%s\n", failures == 0 ? "PASS" : "FAIL");
  return failures == 0 ? 0 : 1;
}
