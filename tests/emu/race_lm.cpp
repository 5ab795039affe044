// The linear recurrence, its gradient, its step and the page calls once each in their forms, for the
// race-detecting build: results are checked elsewhere, here only that no two wavefronts meet in memory.
// (A step with several rows of one slot is left out: the later rows ask for the state before they know
// that they are not the first, and leave without what they read.)
#include <cstdio>
#include <cstdint>
#include <vector>

#include "thrust_cdna4.h"

namespace {

using Words = std::vector<uint64_t>;
int g_failed = 0;

void expect(int rc, const char* what) {
  if (rc != 0) {
    std::printf("%s: %d\n", what, rc);
    g_failed = 1;
  }
}

// both ways; small gates make products leave the range of 32 bits
void scan(int64_t batch, int64_t rows, int64_t channels, const std::vector<int32_t>& offsets, float smallest) {
  const size_t n = (size_t)(batch * rows * channels);
  std::vector<float> gate(n), x(n), out(n), grad_out(n, 1.f), grad_gate(n), grad_x(n);
  for (size_t i = 0; i < n; i++) gate[i] = i % 5 ? 0.5f + 0.04f * (float)(i * 37 % 11) : smallest, x[i] = (float)(i * 13 % 7) - 3.f;
  const int64_t sequences = offsets.empty() ? batch : (int64_t)offsets.size() - 1;
  const size_t states = (size_t)(sequences * channels);
  std::vector<float> init(states, 1.f), final_state(states), grad_final(states, .5f), grad_init(states);
  std::vector<float> chunks((size_t)(batch * ((rows + 63) / 64) * channels));
  thrust_cdna4_linear_scan_args a{};
  a.gate_dtype = a.x_dtype = THRUST_CDNA4_F32;
  a.batch = batch, a.rows = rows, a.channels = channels, a.sequences = sequences;
  a.gate = gate.data(), a.x = x.data(), a.out = out.data();
  a.gate_batch_stride = a.x_batch_stride = a.out_batch_stride = rows * channels;
  a.gate_row_stride = a.x_row_stride = a.out_row_stride = channels;
  a.init = init.data(), a.final_state = final_state.data(), a.states = chunks.data();
  if (!offsets.empty()) a.offsets = offsets.data(), a.offset_bytes = 4, a.clear_outside = 1;
  size_t bytes = 0;
  expect(thrust_cdna4_linear_scan(nullptr, &bytes, &a, nullptr), "linear_scan, size");
  Words temp(bytes / 8 + 1, 0xabcdefull);
  expect(thrust_cdna4_linear_scan(temp.data(), &bytes, &a, nullptr), "linear_scan");
  thrust_cdna4_linear_scan_backward_args b{};
  b.gate_dtype = b.x_dtype = THRUST_CDNA4_F32;
  b.batch = batch, b.rows = rows, b.channels = channels, b.sequences = sequences;
  b.gate = gate.data(), b.x = x.data(), b.grad_out = grad_out.data(), b.grad_gate = grad_gate.data(), b.grad_x = grad_x.data();
  b.gate_batch_stride = b.x_batch_stride = b.grad_out_batch_stride = b.grad_gate_batch_stride = b.grad_x_batch_stride = rows * channels;
  b.gate_row_stride = b.x_row_stride = b.grad_out_row_stride = b.grad_gate_row_stride = b.grad_x_row_stride = channels;
  b.offsets = a.offsets, b.offset_bytes = a.offset_bytes, b.clear_outside = a.clear_outside;
  b.init = init.data(), b.states = chunks.data(), b.grad_final = grad_final.data(), b.grad_init = grad_init.data();
  expect(thrust_cdna4_linear_scan_backward(nullptr, &bytes, &b, nullptr), "linear_scan_backward, size");
  temp.assign(bytes / 8 + 1, 0x1234);
  expect(thrust_cdna4_linear_scan_backward(temp.data(), &bytes, &b, nullptr), "linear_scan_backward");
}

void step(int64_t batch, int64_t channels) {
  std::vector<float> gate((size_t)(batch * channels), .5f), x(gate.size(), 1.f), out(gate.size()), state(gate.size(), 1.f);
  std::vector<int32_t> slots((size_t)batch);
  for (int64_t i = 0; i < batch; i++) slots[(size_t)i] = (int32_t)(batch - i);  // the first one is out of range
  expect(thrust_cdna4_linear_scan_step(THRUST_CDNA4_F32, THRUST_CDNA4_F32, 0, gate.data(), channels, x.data(), channels, out.data(), channels,
                                       state.data(), batch, slots.data(), batch, channels, nullptr), "linear_scan_step");
}

void pages(int num_pages, int requests) {
  const int sequences = 300, most = 6, width = 8;
  std::vector<float> pool((size_t)num_pages * width, 1.f);
  const uint64_t address = (uint64_t) reinterpret_cast<uintptr_t>(pool.data());
  std::vector<int32_t> tables((size_t)sequences * most, -1), lengths((size_t)sequences, 0), refs((size_t)num_pages, 0);
  const thrust_cdna4_page_cache cache{&address, width * 4, 1, num_pages, 16, sequences, most, tables.data(), lengths.data(), refs.data()};
  std::vector<int32_t> ids((size_t)requests), want(ids), parents(ids), children(ids);
  std::vector<uint8_t> done((size_t)requests);
  for (int i = 0; i < requests; i++) {
    ids[(size_t)i] = i, want[(size_t)i] = i * 29 % 80, parents[(size_t)i] = i % 7, children[(size_t)i] = 100 + i;
  }
  size_t bytes = 0;
  Words temp;
  auto resize = [&](const std::vector<int32_t>& who) {
    expect(thrust_cdna4_pages_resize(nullptr, &bytes, &cache, nullptr, nullptr, requests, nullptr, nullptr), "resize, size");
    temp.assign(bytes / 8 + 1, 77);
    expect(thrust_cdna4_pages_resize(temp.data(), &bytes, &cache, who.data(), want.data(), requests, done.data(), nullptr), "resize");
  };
  resize(ids);
  for (int share = 1; share >= 0; share--) {
    expect(thrust_cdna4_pages_fork(nullptr, &bytes, &cache, nullptr, nullptr, requests, share, nullptr, nullptr), "fork, size");
    temp.assign(bytes / 8 + 1, 5);
    expect(thrust_cdna4_pages_fork(temp.data(), &bytes, &cache, parents.data(), children.data(), requests, share, done.data(), nullptr), "fork");
    if (share) {  // cut back into what they share, and grown again
      for (int add = 0; add < 2; add++) {
        for (int i = 0; i < requests; i++) want[(size_t)i] = 5 + add;
        resize(children);
      }
    }
    expect(thrust_cdna4_pages_free(&cache, children.data(), requests, done.data(), nullptr), "free");
  }
  int32_t live = 0;
  expect(thrust_cdna4_pages_compact(nullptr, &bytes, &cache, nullptr, nullptr, nullptr, nullptr), "compact, size");
  temp.assign(bytes / 8 + 1, 9);
  expect(thrust_cdna4_pages_compact(temp.data(), &bytes, &cache, tables.data(), refs.data(), &live, nullptr), "compact");
}

}  // namespace

int main() {
  scan(1, 700, 3, {}, 0.5f);
  scan(2, 300, 132, {}, 1e-20f);
  scan(1, 700, 132, {0, 3, 3, 500, 690}, 0.f);
  scan(1, 5000, 1, {}, 0.9f);
  step(3, 70);
  step(40, 1030);
  for (int num_pages : {100, 9000}) {
    for (int requests : {5, 90}) pages(num_pages, requests);
  }
  std::printf("race_lm: %s\n", g_failed ? "failed" : "done");
  return g_failed;
}
