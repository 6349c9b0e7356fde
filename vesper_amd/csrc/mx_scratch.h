// A context's scratch: a buffer that grows, and what it was before where a captured graph may still use it. Plain C++, also
// built for the CPU, where its steps are tested.
#pragma once
#include <cstdint>
#include <new>

namespace mxs {

struct Kept {
  void* p;
  Kept* next;
};

struct Scratch {
  void* p = nullptr;
  uint64_t bytes = 0;
  bool held = false;      // a call under stream capture was given p: its graph may be replayed until the context closes
  Kept* kept = nullptr;   // earlier buffers of which that is so
};

// At least `bytes` for a call whose stream is captured or not. alloc(&p, bytes) and release(p) return 0 or a status, which
// goes back to the caller. A buffer that a capture was given is never released here, and none is while a stream is captured.
template <typename Alloc, typename Release>
int reserve(Scratch& s, uint64_t bytes, bool capturing, Alloc alloc, Release release, int no_memory) {
  if (s.bytes < bytes) {
    if (s.p && (s.held || capturing)) {
      Kept* entry = new (std::nothrow) Kept{s.p, s.kept};
      if (!entry) return no_memory;
      void* p = nullptr;
      if (int status = alloc(&p, bytes)) {
        delete entry;
        return status;
      }
      s.kept = entry, s.p = p, s.bytes = bytes, s.held = false;
    } else {
      if (s.p)
        if (int status = release(s.p)) return status;
      s.p = nullptr, s.bytes = 0;
      if (int status = alloc(&s.p, bytes)) return status;
      s.bytes = bytes;
    }
  }
  s.held |= capturing;
  return 0;
}

template <typename Release>
void release_all(Scratch& s, Release release) {
  if (s.p) release(s.p);
  while (s.kept) {
    Kept* entry = s.kept;
    s.kept = entry->next;
    release(entry->p);
    delete entry;
  }
  s = Scratch();
}

}  // namespace mxs
