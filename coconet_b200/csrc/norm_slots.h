// Device memory for the partial sums of gradient norms at world size 1.  Two norms
// that run at once must not share any, so every stream has its own slot, and so has
// every captured call, for as long as the graph it was captured into lives (its
// executable graphs included).
#pragma once

#include <cuda_runtime.h>

#include <map>
#include <memory>
#include <mutex>
#include <vector>

#include "list_step.cuh"

namespace coco {

class NormSlots : public std::enable_shared_from_this<NormSlots> {
 public:
  // ctas: the most that a call has.
  explicit NormSlots(int ctas) {
    slot_bytes_ = (sizeof(NormSlot) + sizeof(double) * (size_t)ctas + 127) / 128 * 128;
  }

  // The slot of the next norm on `stream`; the device is current.
  cudaError_t of(cudaStream_t stream, NormSlot **out) {
    std::lock_guard<std::mutex> lock(mu_);
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    cudaGraph_t graph = nullptr;
    unsigned long long id = 0;
    cudaError_t e = cudaStreamGetCaptureInfo(stream, &status, &id, &graph, nullptr, nullptr);
    if (e != cudaSuccess) return e;
    if (status == cudaStreamCaptureStatusInvalidated) return cudaErrorStreamCaptureInvalidated;
    if (status == cudaStreamCaptureStatusActive) return captured(graph, out);
    // the id, unlike the handle, is never used again for another stream
    if ((e = cudaStreamGetId(stream, &id)) != cudaSuccess) return e;
    const auto at = by_stream_.find(id);
    if (at != by_stream_.end()) {
      *out = at->second;
      return cudaSuccess;
    }
    if (by_stream_.size() >= kMaxStreams && (e = forget_streams()) != cudaSuccess) return e;
    if ((e = take(out)) != cudaSuccess) return e;
    by_stream_[id] = *out;
    return cudaSuccess;
  }

  // The communicator goes; nothing runs on the device any more.  (Graphs that still
  // live give their slots back to an empty pool.)
  void destroy() {
    std::lock_guard<std::mutex> lock(mu_);
    for (char *c : chunks_) cudaFree(c);
    if (fill_) cudaStreamDestroy(fill_);
    chunks_.clear(), free_.clear(), by_stream_.clear();
    fill_ = nullptr;
    std::lock_guard<std::mutex> lock_back(back_mu_);
    back_.clear(), closed_ = true;
  }

  cudaError_t grow() {  // by one chunk; allowed while a stream is being captured
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return e;
    char *chunk = nullptr;
    e = fill_ ? cudaSuccess : cudaStreamCreateWithFlags(&fill_, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMalloc((void **)&chunk, slot_bytes_ * kChunk);
    if (e == cudaSuccess) e = cudaMemsetAsync(chunk, 0, slot_bytes_ * kChunk, fill_);
    if (e == cudaSuccess) e = cudaStreamSynchronize(fill_);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
      if (chunk) cudaFree(chunk);
      return e;
    }
    chunks_.push_back(chunk);
    {
      std::lock_guard<std::mutex> lock_back(back_mu_);
      back_.reserve(chunks_.size() * kChunk);  // giving one back allocates nothing
    }
    for (int k = kChunk - 1; k >= 0; --k) free_.push_back((NormSlot *)(chunk + slot_bytes_ * k));
    return cudaSuccess;
  }

 private:
  static constexpr int kChunk = 64;
  static constexpr size_t kMaxStreams = 256;  // remembered; a program that makes one per step stays bounded

  struct Captured {
    std::shared_ptr<NormSlots> owner;
    NormSlot *slot;
  };
  // The last graph that holds the call is gone, and its launches have finished: the
  // runtime keeps the object until then.  Runs on a thread of the runtime and so takes
  // no lock that is held across calls into it.
  static void CUDART_CB give_back(void *p) {
    std::unique_ptr<Captured> c((Captured *)p);
    std::lock_guard<std::mutex> lock_back(c->owner->back_mu_);
    if (!c->owner->closed_) c->owner->back_.push_back(c->slot);
  }

  cudaError_t take(NormSlot **out) {
    {
      std::lock_guard<std::mutex> lock_back(back_mu_);
      free_.insert(free_.end(), back_.begin(), back_.end());
      back_.clear();
    }
    if (free_.empty()) {
      const cudaError_t e = grow();
      if (e != cudaSuccess) return e;
    }
    *out = free_.back();
    free_.pop_back();
    return cudaSuccess;
  }
  cudaError_t captured(cudaGraph_t graph, NormSlot **out) {
    auto c = std::make_unique<Captured>(Captured{shared_from_this(), nullptr});
    cudaError_t e = take(out);
    if (e != cudaSuccess) return e;
    c->slot = *out;
    cudaUserObject_t object = nullptr;
    e = cudaUserObjectCreate(&object, c.get(), give_back, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) {
      free_.push_back(*out);
      return e;
    }
    c.release();  // the object's now; if the graph does not take it, the slot stays unused
    return cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
  }
  // Every norm of a stream so far has finished when the device has.
  cudaError_t forget_streams() {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return e;
    e = cudaDeviceSynchronize();
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return e;
    for (const auto &kv : by_stream_) free_.push_back(kv.second);
    by_stream_.clear();
    return cudaSuccess;
  }

  std::mutex mu_;
  size_t slot_bytes_;
  std::vector<char *> chunks_;
  std::vector<NormSlot *> free_;
  std::map<unsigned long long, NormSlot *> by_stream_;
  cudaStream_t fill_ = nullptr;
  std::mutex back_mu_;            // of what follows; taken last
  std::vector<NormSlot *> back_;  // slots of graphs that are gone
  bool closed_ = false;
};

}  // namespace coco
