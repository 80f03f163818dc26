// Host-only check of the lists' staging slots (yafsdp_amd/csrc/stage_slots.h).  Test infrastructure: no GPU, no HIP.
//
// Host threads claim slots, fill them and queue them on streams; a thread that plays the GPU takes the streams' queues
// in a random order, reads each piece of a slot some time after it was queued and then stores its done word.  Checked:
//   * what the GPU reads is what the claiming thread wrote (nobody refilled the slot before it was read);
//   * a claim of a fitting size fails only while all slots are out, and an oversized or empty one always does;
//   * an abandoned slot can be claimed again.
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <chrono>
#include <deque>
#include <random>
#include <thread>
#include <vector>

#include "../../yafsdp_amd/csrc/stage_slots.h"

using yafsdp::StageSlots;

struct Job {
  int slot;
  uint32_t number, seed;
  size_t bytes;
};

static void fail(const char* what) {
  printf("FAILED: %s\n", what);
  exit(1);
}

static uint32_t word(uint32_t seed, size_t i) { return seed * 2654435761u + uint32_t(i) * 40503u; }

int main() {
  alignas(16) static char block[StageSlots::kBlockBytes];
  static StageSlots slots;
  if (slots.attached()) fail("attached before attach");
  slots.attach(block);

  // single-threaded: exhaustion, sizes, abandon
  uint32_t n = 0;
  if (slots.claim(0, &n) != -1 || slots.claim(StageSlots::kSlotBytes + 1, &n) != -1) fail("sizes that do not fit");
  std::vector<int> held;
  std::vector<uint32_t> numbers;
  for (int i = 0; i < StageSlots::kSlots; i++) {
    const int s = slots.claim(StageSlots::kPieceBytes + 1, &n);
    if (s < 0 || n == 0) fail("a free slot was refused");
    for (int other : held)
      if (other == s) fail("a slot was handed out twice");
    held.push_back(s);
    numbers.push_back(n);
  }
  if (slots.claim(16, &n) != -1) fail("a slot was handed out while all are unread");
  slots.done(held[3])[0].store(numbers[3]);  // one of two pieces: not free yet
  if (slots.claim(16, &n) != -1) fail("a half-read slot was handed out");
  slots.done(held[3])[1].store(numbers[3]);
  if (slots.claim(16, &n) != held[3]) fail("the read slot was not handed out");
  slots.abandon(held[3]);
  if (slots.claim(16, &n) != held[3]) fail("the abandoned slot was not handed out");
  slots.abandon(held[3]);
  for (int i = 0; i < StageSlots::kSlots; i++)
    for (int p = 0; p < 2 && i != 3; p++) slots.done(held[i])[p].store(numbers[i]);

  // threads
  constexpr int kStreams = 5, kHosts = 4, kCalls = 600;
  std::deque<Job> queue[kStreams];
  std::mutex queues;
  std::atomic<int> hosts_left{kHosts};
  std::atomic<long> refused{0}, served{0};
  std::vector<std::thread> hosts;
  for (int h = 0; h < kHosts; h++)
    hosts.emplace_back([&, h] {
      std::mt19937 rng(h);
      for (int c = 0; c < kCalls; c++) {
        const size_t bytes = 16 * (1 + rng() % (c % 7 ? 3000 : StageSlots::kSlotBytes / 16));
        Job j{-1, 0, uint32_t(rng()), bytes};
        for (;;) {
          {
            std::lock_guard<std::mutex> lock(slots.mutex);
            j.slot = slots.claim(bytes, &j.number);
          }
          if (j.slot >= 0) break;
          refused++;
          std::this_thread::sleep_for(std::chrono::microseconds(20));
        }
        uint32_t* w = reinterpret_cast<uint32_t*>(slots.data(j.slot));
        for (size_t i = 0; i < bytes / 4; i++) w[i] = word(j.seed, i);
        if (rng() % 50 == 0) {
          std::lock_guard<std::mutex> lock(slots.mutex);
          slots.abandon(j.slot);
          continue;
        }
        std::lock_guard<std::mutex> lock(queues);
        queue[rng() % kStreams].push_back(j);
      }
      hosts_left--;
    });
  std::thread gpu([&] {
    std::mt19937 rng(99);
    for (;;) {
      Job j{-1, 0, 0, 0};
      bool empty = true;
      {
        std::lock_guard<std::mutex> lock(queues);
        for (auto& q : queue) empty = empty && q.empty();
        auto& q = queue[rng() % kStreams];
        if (!q.empty()) {
          j = q.front();
          q.pop_front();
        }
      }
      if (j.slot < 0) {
        if (empty && hosts_left == 0) return;
        continue;
      }
      if (rng() % 8 == 0) std::this_thread::sleep_for(std::chrono::microseconds(50));
      const uint32_t* w = reinterpret_cast<const uint32_t*>(slots.data(j.slot));
      const int pieces = StageSlots::pieces(j.bytes), from = int(rng() % pieces);
      for (int k = 0; k < pieces; k++) {
        const int p = (from + k) % pieces;
        const size_t end = j.bytes < (p + 1) * StageSlots::kPieceBytes ? j.bytes : (p + 1) * StageSlots::kPieceBytes;
        for (size_t i = p * StageSlots::kPieceBytes / 4; i < end / 4; i++)
          if (w[i] != word(j.seed, i)) fail("the GPU read something else than was staged");
        slots.done(j.slot)[p].store(j.number, std::memory_order_release);
      }
      served++;
    }
  });
  for (auto& t : hosts) t.join();
  gpu.join();
  for (int i = 0; i < StageSlots::kSlots; i++)
    if (slots.claim(16, &n) < 0) fail("a slot was lost");
  printf("ok: %ld served, %ld refused\n", served.load(), refused.load());
  return served > 1000 ? 0 : 1;
}
