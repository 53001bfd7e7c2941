/* A stand-in for the HIP runtime on a machine without a GPU (tests/test_tree_device.py preloads
 * it): two devices, allocations that are counted and can be made to fail, launches that are
 * recorded and run nothing, and the thread's last error. */
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

typedef struct { uint32_t x, y, z; } Dim;

static int device, last;
static int64_t used, room = INT64_MAX, launches, failing;
static struct { Dim grid, block; size_t shared; void* stream; } config;
static int64_t grid_x, block_x;

static int fail(int e) { last = e; return e; }

int hipGetDevice(int* d) { *d = device; return 0; }
int hipSetDevice(int d) {
  if (d < 0 || d > 1) return fail(101);
  device = d;
  return 0;
}
int hipGetLastError(void) { const int e = last; last = 0; return e; }
int hipDeviceGetAttribute(int* v, int what, int d) { (void)what; (void)d; *v = 0; return 0; }
int hipMalloc(void** p, size_t n) {
  if (used > room - (int64_t)n) return failing++, fail(2);
  used += (int64_t)n;
  size_t* q = malloc(sizeof(size_t));
  *q = n;
  *p = q;
  return 0;
}
int hipFree(void* p) {
  if (!p) return 0;
  used -= (int64_t)*(size_t*)p;
  free(p);
  return 0;
}
int hipMemset(void* p, int v, size_t n) { (void)p; (void)v; (void)n; return 0; }
int hipMemcpy(void* to, const void* from, size_t n, int kind) { (void)from; (void)kind; memset(to, 0, n); return 0; }
int hipGetSymbolAddress(void** p, const void* s) { (void)s; *p = 0; return fail(13); }
int hipDeviceSynchronize(void) { return 0; }
int hipStreamSynchronize(void* s) { (void)s; return 0; }
int __hipPushCallConfiguration(Dim g, Dim b, size_t shared, void* stream) {
  config.grid = g;
  config.block = b;
  config.shared = shared;
  config.stream = stream;
  return 0;
}
int __hipPopCallConfiguration(Dim* g, Dim* b, size_t* shared, void** stream) {
  *g = config.grid;
  *b = config.block;
  *shared = config.shared;
  *stream = config.stream;
  return 0;
}
int hipLaunchKernel(const void* f, Dim g, Dim b, void** args, size_t shared, void* stream) {
  (void)f; (void)args; (void)shared; (void)stream;
  launches++;
  grid_x = g.x;
  block_x = b.x;
  return 0;
}

/* what the tests ask */
int fake_last_error(void) { return last; }
int64_t fake_used(void) { return used; }
int64_t fake_launches(void) { return launches; }
int64_t fake_work_items(void) { return grid_x * block_x; }
void fake_room(int64_t n) { room = n; }
