/* The few HIP calls that a launch makes, written down instead of made: loaded before libposehip.so, so that a process without
 * a GPU can see which kernel a call would launch, with which grid and how much LDS. */
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#include <unistd.h>

typedef struct { uint32_t x, y, z; } dim;
typedef struct {
  const char* name;   /* of the kernel; NULL: not registered */
  int64_t what;       /* 0: launch, 1: the largest dynamic LDS is set */
  int64_t grid[3], block[3], lds;
  int64_t most;       /* a launch: dynamic LDS that its kernel may have */
} call;

#define N 4096
static struct { const void* fn; const char* name; int64_t most; } fns[N];
static call calls[N];
static int n_fns, n_calls, device;
static volatile int wait_ms, setters;
static __thread struct { dim g, b; size_t lds; void* st; } pushed;

static call* next(const void* fn, int what) {
  static call full;
  const int at = __atomic_fetch_add(&n_calls, 1, __ATOMIC_SEQ_CST);
  call* c = at < N ? &calls[at] : &full;
  memset(c, 0, sizeof *c);
  c->what = what;
  for (int i = 0; i < n_fns; i++)
    if (fns[i].fn == fn) c->name = fns[i].name, c->most = fns[i].most;
  return c;
}

int fake_calls(void) { return n_calls < N ? n_calls : N; }
const call* fake_call(int i) { return &calls[i]; }
void fake_clear(void) { n_calls = 0; }
/* whoever sets a largest LDS first waits for the next to do so, this long at the most */
void fake_wait(int ms) { setters = 0, wait_ms = ms; }
int fake_setters(void) { return setters; }

void** __hipRegisterFatBinary(const void* data) { static void* handle; return &handle; }
void __hipUnregisterFatBinary(void** modules) {}
void __hipRegisterFunction(void** modules, const void* fn, char* device_fn, const char* name, unsigned threads, void* tid, void* bid,
                           void* block, void* grid, int* size) {
  if (n_fns < N) fns[n_fns].fn = fn, fns[n_fns].most = 65536, fns[n_fns++].name = strdup(name);
}
void __hipRegisterVar(void** modules, void* var, char* host, char* name, int ext, size_t size, int constant, int global) {}
int __hipPushCallConfiguration(dim g, dim b, size_t lds, void* st) {
  pushed.g = g, pushed.b = b, pushed.lds = lds, pushed.st = st;
  return 0;
}
int __hipPopCallConfiguration(dim* g, dim* b, size_t* lds, void** st) {
  *g = pushed.g, *b = pushed.b, *lds = pushed.lds, *st = pushed.st;
  return 0;
}
int hipGetDevice(int* d) { *d = device; return 0; }
int hipSetDevice(int d) { device = d; return 0; }
int hipGetLastError(void) { return 0; }
int hipFuncSetAttribute(const void* fn, int attr, int value) {
  next(fn, 1)->lds = value;
  for (int i = 0; i < n_fns; i++)
    if (fns[i].fn == fn) fns[i].most = value;
  if (__atomic_add_fetch(&setters, 1, __ATOMIC_SEQ_CST) == 1)
    for (int ms = 0; ms < wait_ms && setters < 2; ms++) usleep(1000);
  return 0;
}
int hipLaunchKernel(const void* fn, dim g, dim b, void** args, size_t lds, void* st) {
  call* c = next(fn, 0);
  c->grid[0] = g.x, c->grid[1] = g.y, c->grid[2] = g.z;
  c->block[0] = b.x, c->block[1] = b.y, c->block[2] = b.z;
  c->lds = (int64_t)lds;
  return 0;
}
