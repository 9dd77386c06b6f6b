// What a captured call uses beside its arguments (counters, a status word) has to be there for as long as the graph can be replayed, and may be
// given to another call when it cannot any more. The graph itself tells: a user object goes with it, into every executable made of it, and
// is destroyed with the last of these, not before a replay under way has ended. Its destructor may not call CUDA, so it leaves a note here.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <vector>

#include "eux_kernels.h"

namespace eux {

struct GraphNotes {
  std::mutex lock;
  std::vector<uint64_t> gone;  // with room for all that are held: the destructor must not fail
  size_t held = 0;
};
static GraphNotes& graph_notes() {
  static GraphNotes* const notes = new GraphNotes;  // never destroyed: graphs may be, while the process ends
  return *notes;
}
static void CUDART_CB graph_is_gone(void* token) {
  GraphNotes& notes = graph_notes();
  std::lock_guard<std::mutex> lock(notes.lock);
  notes.gone.push_back((uint64_t)(uintptr_t)token);
  --notes.held;
}

}  // namespace eux

using namespace eux;

extern "C" int eux_graph_hold(void* stream, uint64_t token) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  if (cudaError_t e = cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &id, &graph); e != cudaSuccess) return (int)e;
  if (status != cudaStreamCaptureStatusActive || !graph) return EUX_ERR_BAD_ARG;
  GraphNotes& notes = graph_notes();
  {
    std::lock_guard<std::mutex> lock(notes.lock);
    try {
      const size_t need = notes.gone.size() + notes.held + 1;
      if (notes.gone.capacity() < need) notes.gone.reserve(2 * need);
    } catch (...) {
      return EUX_ERR_TOO_LARGE;
    }
    ++notes.held;
  }
  cudaUserObject_t object;
  if (cudaError_t e = cudaUserObjectCreate(&object, (void*)(uintptr_t)token, graph_is_gone, 1, cudaUserObjectNoDestructorSync); e != cudaSuccess) {
    std::lock_guard<std::mutex> lock(notes.lock);
    --notes.held;
    return (int)e;
  }
  const cudaError_t e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
  if (e != cudaSuccess) cudaUserObjectRelease(object, 1);  // its destructor leaves the note all the same
  return (int)e;
}

extern "C" int eux_graphs_gone(uint64_t* tokens, int most) {
  if (!tokens || most < 0) return 0;
  GraphNotes& notes = graph_notes();
  std::lock_guard<std::mutex> lock(notes.lock);
  const int n = (int)std::min<size_t>(notes.gone.size(), (size_t)most);
  std::copy(notes.gone.end() - n, notes.gone.end(), tokens);
  notes.gone.resize(notes.gone.size() - n);
  return n;
}
