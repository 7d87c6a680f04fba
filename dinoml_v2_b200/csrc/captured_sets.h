// Workspaces of captured work, one set per (device, capture, stream).  A captured launch keeps the addresses that it was captured with and its graph may be replayed on any
// stream, beside other graphs of the same capture stream and beside that stream's own calls; the launches of one stream within one capture are ordered.  So they share a
// set that nobody else has, and that is given back when the graph and everything instantiated from it is gone (a user object of the graph tells).  Replays of one instantiated
// graph are ordered by CUDA.  Host code over the CUDA runtime only.
#pragma once
#include "scratch_sets.h"

namespace b200gguf {

// Within its scope this thread may allocate and wait for streams of its own although a stream is being captured.
class AllocationsDuringCapture {
 public:
  AllocationsDuringCapture() { cudaThreadExchangeStreamCaptureMode(&mode_); }
  ~AllocationsDuringCapture() { cudaThreadExchangeStreamCaptureMode(&mode_); }
  AllocationsDuringCapture(const AllocationsDuringCapture&) = delete;
  AllocationsDuringCapture& operator=(const AllocationsDuringCapture&) = delete;

 private:
  cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
};

// Empties a set at once, on a stream that is in no capture.
template <typename Set> inline bool empty_now(Set& set) {
  cudaStream_t s = nullptr;
  if (cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking) != cudaSuccess) return false;
  const bool emptied = set.empty(s) && cudaStreamSynchronize(s) == cudaSuccess;
  cudaStreamDestroy(s);
  return emptied;
}

template <typename Set>
class CapturedSets {
 public:
  static constexpr size_t kMaxSpare = 4;      // per device
  std::mutex mutex;                           // held by the caller of everything below

  // The set of this capture on this stream, which may not be made() yet; null if it can't be had.  Within AllocationsDuringCapture.
  Set* at(int dev, unsigned long long capture, cudaGraph_t graph, cudaStream_t stream) {
    collect();
    for (Lease* lease : leases_)
      if (lease->dev == dev && lease->capture == capture && lease->stream == stream) return &lease->set;
    Lease* lease = new Lease{this, dev, capture, stream, Set{}};
    std::vector<Set>& spare = spare_[dev];
    if (!spare.empty()) {
      lease->set = std::move(spare.back());
      spare.pop_back();
      if (!empty_now(lease->set)) {             // (a launch of the graph that had it may have given up)
        lease->set.give_back();
        delete lease;
        return nullptr;
      }
    }
    leases_.push_back(lease);
    cudaUserObject_t object = nullptr;
    if (cudaUserObjectCreate(&object, lease, give_back, 1, cudaUserObjectNoDestructorSync) != cudaSuccess) {
      give_back(lease);
      return nullptr;
    }
    if (cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove) != cudaSuccess) {
      cudaUserObjectRelease(object, 1);         // (calls give_back)
      return nullptr;
    }
    return &lease->set;
  }
  // Sets whose graphs are gone become spare ones (a bounded number) or are freed.
  void collect() {
    std::vector<Lease*> gone;
    {
      std::lock_guard<std::mutex> lock(returned_mutex_);
      gone.swap(returned_);
    }
    for (Lease* lease : gone) {
      for (size_t i = 0; i < leases_.size(); ++i)
        if (leases_[i] == lease) { leases_.erase(leases_.begin() + i); break; }
      std::vector<Set>& spare = spare_[lease->dev];
      if (lease->set.made() && spare.size() < kMaxSpare) spare.push_back(std::move(lease->set));
      else lease->set.give_back();
      delete lease;
    }
  }
  // The sets in use on a device are empty when this returns.
  bool empty_all(int dev) {
    bool emptied = true;
    for (Lease* lease : leases_)
      if (lease->dev == dev) emptied = lease->set.empty(nullptr) && emptied;
    return cudaStreamSynchronize(nullptr) == cudaSuccess && emptied;
  }

 private:
  struct Lease {
    CapturedSets* owner;
    int dev;
    unsigned long long capture;
    cudaStream_t stream;
    Set set;
  };
  // From whatever thread drops the last reference, with no CUDA call allowed: `mutex` may be held.
  static void CUDART_CB give_back(void* p) {
    Lease* lease = static_cast<Lease*>(p);
    CapturedSets* owner = lease->owner;
    std::lock_guard<std::mutex> lock(owner->returned_mutex_);
    owner->returned_.push_back(lease);
  }

  std::vector<Lease*> leases_;
  std::map<int, std::vector<Set>> spare_;
  std::mutex returned_mutex_;
  std::vector<Lease*> returned_;
};

// The attention's workspaces: of streams, and of captures.
class AttnWorkspaces {
 public:
  // Room for `floats` of pieces and the counters, for a launch on `stream` of the current device; null if there is none.
  float* get(int dev, cudaStream_t stream, size_t floats, int** arrived) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long capture = 0;
    cudaGraph_t graph = nullptr;
    if (cudaStreamGetCaptureInfo(stream, &status, &capture, &graph, nullptr, nullptr) != cudaSuccess || status == cudaStreamCaptureStatusInvalidated) return nullptr;
    if (status == cudaStreamCaptureStatusActive) {
      std::lock_guard<std::mutex> lock(captured_.mutex);
      AllocationsDuringCapture allowed;
      AttnScratch* set = captured_.at(dev, capture, graph, stream);
      if (set == nullptr || !make(*set, [&] { return empty_now(*set); }) || !grow(*set, floats, floats)) return nullptr;
      *arrived = set->arrived;
      return set->partial;
    }
    std::lock_guard<std::mutex> lock(sets_.mutex);
    AttnScratch& set = sets_.at(dev, stream);
    if (!make(set, [&] { return set.empty(stream); }) || !grow(set, floats, floats > 2 * set.floats ? floats : 2 * set.floats)) return nullptr;
    *arrived = set.arrived;
    return set.partial;
  }
  // `stream` is about to be destroyed and has no work left.
  void release(cudaStream_t stream) {
    std::lock_guard<std::mutex> lock(sets_.mutex);
    sets_.release(stream);
  }
  void reset(int dev) {
    {
      std::lock_guard<std::mutex> lock(sets_.mutex);
      sets_.empty_all(dev);
    }
    std::lock_guard<std::mutex> lock(captured_.mutex);
    captured_.collect();
    captured_.empty_all(dev);
  }

 private:
  template <typename Empty> static bool make(AttnScratch& set, Empty empty) {
    if (set.made()) return true;
    if (cudaMalloc(reinterpret_cast<void**>(&set.arrived), sizeof(int) * AttnScratch::kMaxWorkers) != cudaSuccess) { set.arrived = nullptr; return false; }
    if (empty()) return true;
    cudaFree(set.arrived);
    set.arrived = nullptr;
    return false;
  }
  // Launches that are on their way keep the smaller room.
  static bool grow(AttnScratch& set, size_t floats, size_t size) {
    if (floats <= set.floats) return true;
    float* p = nullptr;
    if (cudaMalloc(reinterpret_cast<void**>(&p), size * sizeof(float)) != cudaSuccess) return false;
    if (set.partial != nullptr) set.outgrown.push_back(set.partial);
    set.partial = p;
    set.floats = size;
    return true;
  }

  ScratchSets<AttnScratch> sets_;
  CapturedSets<AttnScratch> captured_;
};

}  // namespace b200gguf
