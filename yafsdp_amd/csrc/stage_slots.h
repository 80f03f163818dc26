// Pinned staging slots for the lists that do not fit a launch's arguments: host memory that a kernel reads and then
// marks as read.  The state machine only; no HIP in here (list_api.hip allocates the block and launches the kernel,
// tests/c/stage_slots_check.cpp plays the GPU).
//
// A slot is free when every piece of its last use carries that use's number in its `done` word, which the kernel stores
// after it has read the piece.  claim() never waits: with every slot still unread it returns -1 and the caller takes
// its other route.  A slot is claimed under the mutex and filled outside of it; nobody else touches it in between,
// because its done words do not carry the new number yet.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

namespace yafsdp {

class StageSlots {
 public:
  static constexpr int kSlots = 16;
  static constexpr size_t kPieceBytes = 16384;  // one workgroup's share: 16 bytes for each of 1024 lanes
  static constexpr int kPieces = 32;            // of one slot at most (512 KiB: 43,690 ranges, 10,922 of AdamW)
  static constexpr size_t kSlotBytes = kPieceBytes * kPieces;
  static constexpr size_t kBlockBytes = kSlots * kSlotBytes + kSlots * kPieces * sizeof(uint32_t);

  // the pinned block (kBlockBytes, 16-byte aligned); its done words start at 0, the number of no use
  void attach(void* block) {
    base_ = static_cast<char*>(block);
    done_ = reinterpret_cast<std::atomic<uint32_t>*>(base_ + kSlots * kSlotBytes);
    for (int i = 0; i < kSlots * kPieces; i++) done_[i].store(0, std::memory_order_relaxed);
  }
  bool attached() const { return base_ != nullptr; }

  // a free slot for `bytes`, or -1; *number is what the kernel has to store into the slot's done words
  int claim(size_t bytes, uint32_t* number) {
    if (bytes == 0 || bytes > kSlotBytes) return -1;
    for (int i = 0; i < kSlots; i++) {
      const int s = (next_ + i) % kSlots;
      if (!free(s)) continue;
      next_ = (s + 1) % kSlots;
      if (++number_ == 0) number_ = 1;
      *number = number_;
      last_[s] = number_;
      pieces_[s] = pieces(bytes);
      // no kernel is left that would store here; a word of an older, longer use may not pass for this number once the
      // numbers have wrapped
      for (int p = 0; p < pieces_[s]; p++) done(s)[p].store(0, std::memory_order_relaxed);
      return s;
    }
    return -1;
  }
  // the slot's kernel was not launched after all
  void abandon(int s) {
    for (int p = 0; p < pieces_[s]; p++) done(s)[p].store(last_[s], std::memory_order_release);
  }

  char* data(int s) { return base_ + size_t(s) * kSlotBytes; }
  std::atomic<uint32_t>* done(int s) { return done_ + s * kPieces; }
  static int pieces(size_t bytes) { return int((bytes + kPieceBytes - 1) / kPieceBytes); }

  std::mutex mutex;  // held by the caller around attach, claim and abandon

 private:
  bool free(int s) {
    for (int p = 0; p < pieces_[s]; p++)
      if (done(s)[p].load(std::memory_order_acquire) != last_[s]) return false;
    return true;
  }
  char* base_ = nullptr;
  std::atomic<uint32_t>* done_ = nullptr;
  uint32_t number_ = 0;
  uint32_t last_[kSlots] = {};
  int pieces_[kSlots] = {};  // of the slot's last use; 0: never used
  int next_ = 0;
};

}  // namespace yafsdp
