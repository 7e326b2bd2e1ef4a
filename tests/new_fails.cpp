// operator new that fails on demand (LD_PRELOAD): the allocation of exactly
// `size` bytes that follows `skip` others of that size throws std::bad_alloc.
#include <cstdlib>
#include <new>

static thread_local size_t g_size = 0;
static thread_local int g_skip = 0, g_failed = 0;

extern "C" void new_fails_at(size_t size, int skip) { g_size = size, g_skip = skip, g_failed = 0; }
extern "C" int new_failed(void) { return g_failed; }

void *operator new(size_t n) {
  if (g_size != 0 && n == g_size && g_skip-- == 0) {
    g_size = 0, g_failed = 1;
    throw std::bad_alloc();
  }
  if (void *p = std::malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void *operator new[](size_t n) { return operator new(n); }
void operator delete(void *p) noexcept { std::free(p); }
void operator delete[](void *p) noexcept { std::free(p); }
void operator delete(void *p, size_t) noexcept { std::free(p); }
void operator delete[](void *p, size_t) noexcept { std::free(p); }
