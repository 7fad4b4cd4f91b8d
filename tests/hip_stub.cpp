// The HIP runtime's entry points that liblq_seq.so calls, for tests of its host side without a GPU: nothing is launched.
#include <stddef.h>
struct Dim3 { unsigned x, y, z; };
static int device, asked[8], launches, fail;
static Dim3 grid, block;
static size_t lds;
extern "C" {
void stub_device(int d) { device = d; }
void stub_fail(int n) { fail = n; }                  // the next n hipFuncSetAttribute fail
int stub_asked(int d) { return asked[d]; }           // hipFuncSetAttribute on device d that did not
int stub_launches() { return launches; }
int hipGetDevice(int* d) { *d = device; return 0; }
int hipDeviceGetAttribute(int* v, int, int) { *v = 256; return 0; }
int hipFuncSetAttribute(const void*, int, int) {
  if (fail) return --fail, 1;
  return ++asked[device], 0;
}
int hipGetLastError() { return 0; }
int hipLaunchKernel(const void*, Dim3, Dim3, void**, size_t, void*) { return ++launches, 0; }
int __hipPushCallConfiguration(Dim3 g, Dim3 b, size_t l, void*) { return grid = g, block = b, lds = l, 0; }
int __hipPopCallConfiguration(Dim3* g, Dim3* b, size_t* l, void** s) { return *g = grid, *b = block, *l = lds, *s = nullptr, 0; }
void** __hipRegisterFatBinary(const void*) { static void* p; return &p; }
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
void __hipUnregisterFatBinary(void**) {}
}
