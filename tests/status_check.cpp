// Status words of the serving operators: take_status and make_status leave no
// memset behind them that a kernel on a non-blocking stream could overtake.  The
// CUDA runtime is a recorder here: a memset stays pending until a wait.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "sc_serve.h"

static int pending = 0;     // memsets that nothing has waited for
static int word_value = 0;  // the device's word

void sc_set_error(const std::string &) {}

extern "C" {
cudaError_t cudaGetDevice(int *d) { return *d = 0, cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
const char *cudaGetErrorString(cudaError_t) { return ""; }
cudaError_t cudaMalloc(void **p, size_t n) { return *p = std::calloc(1, n), cudaSuccess; }
cudaError_t cudaFree(void *p) { return std::free(p), cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { return pending = 0, cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) { return pending = s ? pending : 0, cudaSuccess; }
cudaError_t cudaMemset(void *p, int v, size_t n) { return std::memset(p, v, n), ++pending, cudaSuccess; }
cudaError_t cudaMemcpy(void *to, const void *from, size_t n, cudaMemcpyKind) { return std::memcpy(to, from, n), cudaSuccess; }
}

#define CHECK(x) if (!(x)) return std::printf("line %d: %s\n", __LINE__, #x), 1

int main() {
  word_value = 8;
  CHECK(sc::serve::take_status(0, &word_value) == 8 && word_value == 0);
  CHECK(pending == 0);
  CHECK(sc::serve::take_status(0, &word_value) == 0 && pending == 0);
  sc::serve::DeviceBlock block;
  sc::serve::make_status(block, 0);
  CHECK(block.p && *static_cast<int *>(block.p) == 0 && pending == 0);
  std::puts("ok");
  return 0;
}
