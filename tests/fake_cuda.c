/* A CUDA runtime without a GPU, for tests of the host code: device memory is
 * host memory, kernels are not run but written down (name, grid, stream,
 * arguments), and a launch can be told to fail. Preloaded into a child
 * process in front of the real runtime.
 *
 * It also watches one rule of the real one: cudaMemcpy from pageable host
 * memory, a device-to-device cudaMemcpy and cudaMemset may return before the
 * device's memory is written, and only the legacy stream orders what follows.
 * A launch or copy on a non-blocking stream before the legacy stream has been
 * waited for is counted in fake_unordered(). */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

typedef int err_t;
typedef struct { unsigned x, y, z; } dim3_t;
enum { INVALID_CONFIGURATION = 9, MAX = 1 << 20 };

/* ---- what the tests ask ---- */
struct launch {
  const char* name;
  dim3_t grid, block;
  void* stream;
  int captured;
};
static struct launch launches[MAX];
static int nlaunches, pending, unordered, last_error;
static char first_unordered[200];
static char fail_name[200];
static int fail_at = -1;
static void* capturing;

int fake_launches(void) { return nlaunches; }
int fake_unordered(void) { return unordered; }
const char* fake_first_unordered(void) { return first_unordered; }
int fake_launch(int i, char* name, int len, unsigned* grid) {
  if (i < 0 || i >= nlaunches) return -1;
  snprintf(name, (size_t)len, "%s", launches[i].name);
  grid[0] = launches[i].grid.x, grid[1] = launches[i].grid.y, grid[2] = launches[i].block.x;
  return 0;
}
/* The n-th launch from now on (0 the next) of a kernel whose name holds
 * `name` is refused. */
void fake_fail(const char* name, int n) {
  snprintf(fail_name, sizeof fail_name, "%s", name);
  fail_at = n;
}

/* ---- kernels ---- */
static const void* fn_ptr[1 << 14];
static const char* fn_name[1 << 14];
static int nfn;
void** __cudaRegisterFatBinary(void* p) {
  (void)p;
  static void* handle;
  return &handle;
}
void __cudaRegisterFatBinaryEnd(void** h) { (void)h; }
void __cudaUnregisterFatBinary(void** h) { (void)h; }
void __cudaRegisterFunction(void** h, const char* host, char* dev, const char* name, int limit, void* tid, void* bid,
                            void* bdim, void* gdim, int* wsize) {
  (void)h, (void)dev, (void)limit, (void)tid, (void)bid, (void)bdim, (void)gdim, (void)wsize;
  if (nfn < 1 << 14) fn_ptr[nfn] = host, fn_name[nfn] = name, nfn++;
}
void __cudaRegisterVar(void** h, char* host, char* dev, const char* name, int ext, size_t size, int constant, int global) {
  (void)h, (void)host, (void)dev, (void)name, (void)ext, (void)size, (void)constant, (void)global;
}
static __thread struct { dim3_t grid, block; size_t smem; void* stream; } config;
unsigned __cudaPushCallConfiguration(dim3_t grid, dim3_t block, size_t smem, void* stream) {
  config.grid = grid, config.block = block, config.smem = smem, config.stream = stream;
  return 0;
}
err_t __cudaPopCallConfiguration(dim3_t* grid, dim3_t* block, size_t* smem, void* stream) {
  *grid = config.grid, *block = config.block, *smem = config.smem, *(void**)stream = config.stream;
  return 0;
}

static void used(void* stream, const char* by) {
  if (stream == NULL || !pending || capturing) return;
  if (!unordered++) snprintf(first_unordered, sizeof first_unordered, "%s", by);
}
static err_t launched(const void* f, dim3_t grid, dim3_t block, void* stream) {
  const char* name = "?";
  for (int i = 0; i < nfn; i++)
    if (fn_ptr[i] == f) name = fn_name[i];
  if (fail_at >= 0 && strstr(name, fail_name) && fail_at-- == 0) return last_error = INVALID_CONFIGURATION;
  used(stream, name);
  if (nlaunches < MAX) {
    struct launch l = {name, grid, block, stream, capturing != NULL};
    launches[nlaunches++] = l;
  }
  return 0;
}
err_t cudaLaunchKernel(const void* f, dim3_t grid, dim3_t block, void** args, size_t smem, void* stream) {
  (void)args, (void)smem;
  return launched(f, grid, block, stream);
}
err_t cudaLaunchCooperativeKernel(const void* f, dim3_t grid, dim3_t block, void** args, size_t smem, void* stream) {
  (void)args, (void)smem;
  return launched(f, grid, block, stream);
}
struct config { dim3_t grid, block; size_t smem; void* stream; void* attrs; unsigned n; };
err_t cudaLaunchKernelExC(const struct config* c, const void* f, void** args) {
  (void)args;
  return launched(f, c->grid, c->block, c->stream);
}

/* ---- memory ---- */
static struct { char* p; size_t n; int device; } blocks[MAX];
static int nblocks;
static err_t take(void** p, size_t n, int device) {
  *p = calloc(n ? n : 1, 1);
  if (!*p) return last_error = 2;
  if (nblocks < MAX) blocks[nblocks].p = *p, blocks[nblocks].n = n, blocks[nblocks].device = device, nblocks++;
  return 0;
}
static int pageable(const void* p) {
  for (int i = nblocks - 1; i >= 0; i--)
    if ((const char*)p >= blocks[i].p && (const char*)p < blocks[i].p + blocks[i].n) return 0;
  return 1;
}
static err_t drop(void* p) {
  for (int i = nblocks - 1; i >= 0; i--)
    if (blocks[i].p == p) {
      blocks[i] = blocks[--nblocks];
      break;
    }
  free(p);
  return 0;
}
err_t cudaMalloc(void** p, size_t n) { return take(p, n, 1); }
err_t cudaFree(void* p) { return drop(p); }
err_t cudaHostAlloc(void** p, size_t n, unsigned flags) { return (void)flags, take(p, n, 0); }
err_t cudaFreeHost(void* p) { return drop(p); }
err_t cudaMemcpy(void* dst, const void* src, size_t n, int kind) { /* kind 1: to the device, 2: from it, 3: on it */
  memmove(dst, src, n);
  if (kind == 2)
    pending = 0; /* behind everything on the legacy stream, and waited for */
  else if (kind == 3 || pageable(src))
    pending = 1;
  return 0;
}
err_t cudaMemcpyAsync(void* dst, const void* src, size_t n, int kind, void* stream) {
  (void)kind;
  used(stream, "cudaMemcpyAsync");
  if (!capturing) memmove(dst, src, n);
  return 0;
}
err_t cudaMemcpy2DAsync(void* dst, size_t dp, const void* src, size_t sp, size_t w, size_t h, int kind, void* stream) {
  (void)kind;
  used(stream, "cudaMemcpy2DAsync");
  for (size_t i = 0; i < h && !capturing; i++) memmove((char*)dst + i * dp, (const char*)src + i * sp, w);
  return 0;
}
err_t cudaMemset(void* p, int v, size_t n) {
  memset(p, v, n);
  pending = 1;
  return 0;
}
err_t cudaMemsetAsync(void* p, int v, size_t n, void* stream) {
  used(stream, "cudaMemsetAsync");
  if (!capturing) memset(p, v, n);
  return 0;
}
static char symbol[1 << 22];
err_t cudaGetSymbolAddress(void** p, const void* s) { return (void)s, *p = symbol, 0; }
err_t cudaMemcpyFromSymbol(void* dst, const void* s, size_t n, size_t off, int kind) {
  (void)s, (void)off, (void)kind;
  memset(dst, 0, n);
  return 0;
}

/* ---- devices, streams, graphs ---- */
err_t cudaGetDeviceCount(int* n) { return *n = 1, 0; }
err_t cudaGetDevice(int* d) { return *d = 0, 0; }
err_t cudaSetDevice(int d) { return d ? (last_error = 101) : 0; }
err_t cudaDeviceGetAttribute(int* v, int attr, int d) {
  (void)d;
  *v = attr == 16 ? 148 : attr == 95 ? 1 : 0; /* multiprocessors; cooperative launches */
  return 0;
}
err_t cudaDeviceSynchronize(void) { return pending = 0, 0; }
err_t cudaFuncSetAttribute(const void* f, int a, int v) { return (void)f, (void)a, (void)v, 0; }
err_t cudaGetLastError(void) {
  const err_t e = last_error;
  last_error = 0;
  return e;
}
err_t cudaPeekAtLastError(void) { return last_error; }
const char* cudaGetErrorString(err_t e) { return e == INVALID_CONFIGURATION ? "invalid configuration argument" : "error"; }
static err_t encode() { return 0; }
err_t cudaGetDriverEntryPoint(const char* s, void** fn, unsigned long long flags, int* found) {
  (void)s, (void)flags;
  *fn = (void*)encode;
  if (found) *found = 0;
  return 0;
}
err_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void* f, int b, size_t s, unsigned flags) {
  return (void)f, (void)b, (void)s, (void)flags, *n = 1, 0;
}
err_t cudaOccupancyMaxActiveClusters(int* n, const void* f, const void* c) { return (void)f, (void)c, *n = 8, 0; }
err_t cudaStreamCreateWithFlags(void** s, unsigned flags) {
  (void)flags;
  *s = malloc(1);
  return 0;
}
err_t cudaStreamDestroy(void* s) { return free(s), 0; }
err_t cudaStreamSynchronize(void* s) {
  if (s == NULL || s == (void*)1) pending = 0;
  return 0;
}
err_t cudaStreamWaitEvent(void* s, void* e, unsigned f) { return (void)s, (void)e, (void)f, 0; }
err_t cudaStreamBeginCapture(void* s, int mode) { return (void)mode, capturing = s, 0; }
err_t cudaStreamEndCapture(void* s, void** g) { return (void)s, capturing = NULL, *g = malloc(1), 0; }
err_t cudaGraphInstantiate(void** x, void* g, unsigned long long f) { return (void)g, (void)f, *x = malloc(1), 0; }
err_t cudaGraphLaunch(void* x, void* s) { return (void)x, used(s, "cudaGraphLaunch"), 0; }
err_t cudaGraphDestroy(void* g) { return free(g), 0; }
err_t cudaGraphExecDestroy(void* x) { return free(x), 0; }
err_t cudaEventCreateWithFlags(void** e, unsigned f) { return (void)f, *e = malloc(1), 0; }
err_t cudaEventDestroy(void* e) { return free(e), 0; }
err_t cudaEventRecord(void* e, void* s) { return (void)e, (void)s, 0; }
err_t cudaEventSynchronize(void* e) { return (void)e, 0; }
