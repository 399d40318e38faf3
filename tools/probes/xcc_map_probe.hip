// Probe: which XCD (XCC_ID) and when a workgroup of a 1-D grid runs -- the assumption behind the "XCD-contiguous
// band" remaps of the tile kernels (t = (b & 7) * (T / 8) + (b >> 3): blockIdx b is dispatched to XCD b % 8).
// build: hipcc --offload-arch=gfx950 -O3 -Xclang -target-feature -Xclang -packed-fp32-ops -o tools/probes/xcc_map_probe tools/probes/xcc_map_probe.hip
#include <hip/hip_runtime.h>
#include <cstdio>
#include <vector>
#define CK(x) do { hipError_t e = (x); if (e != hipSuccess) { printf("HIP error %s at %d\n", hipGetErrorString(e), __LINE__); return 1; } } while (0)
__global__ __launch_bounds__(512) void probe(unsigned* out, int spin) {
  __shared__ float pad[8192];  // 32 KB like fr_forward_nhwc_occ's tiles
  unsigned xcc, hwid;
  asm volatile("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID)" : "=s"(xcc));
  asm volatile("s_getreg_b32 %0, hwreg(HW_REG_HW_ID)" : "=s"(hwid));
  const unsigned long long t0 = __builtin_amdgcn_s_memtime();
  pad[threadIdx.x] = (float)threadIdx.x;
  __syncthreads();
  float acc = 0.f;
  for (int i = 0; i < spin; i++) acc += pad[(threadIdx.x + i) & 8191];
  if (acc == 12345.678f) out[0] = 1;
  if (threadIdx.x == 0) {
    out[blockIdx.x * 4 + 0] = xcc & 0xf;
    out[blockIdx.x * 4 + 1] = hwid;
    out[blockIdx.x * 4 + 2] = (unsigned)(t0 & 0xffffffffu);
    out[blockIdx.x * 4 + 3] = (unsigned)(__builtin_amdgcn_s_memtime() & 0xffffffffu);
  }
}
int main() {
  const int T = 2112;
  unsigned* d; CK(hipMalloc(&d, T * 16)); CK(hipMemset(d, 0, T * 16));
  for (int it = 0; it < 2; it++) { hipLaunchKernelGGL(probe, dim3(T), dim3(512), 0, 0, d, 4000); CK(hipDeviceSynchronize()); }
  std::vector<unsigned> h(T * 4); CK(hipMemcpy(h.data(), d, T * 16, hipMemcpyDeviceToHost));
  int agree = 0; int hist[16] = {0};
  for (int b = 0; b < T; b++) { agree += (int)h[b * 4] == (b & 7); hist[h[b * 4] & 15]++; }
  printf("blocks whose XCC_ID == blockIdx %% 8: %d of %d\n", agree, T);
  printf("blocks per XCC:"); for (int x = 0; x < 8; x++) printf(" %d", hist[x]); printf("\n");
  printf("first 32 blocks (blockIdx: xcc):"); for (int b = 0; b < 32; b++) printf(" %d:%u", b, h[b * 4]); printf("\n");
  // start order inside XCC 0: which blockIdx start, in time order
  unsigned t_min = 0xffffffffu; for (int b = 0; b < T; b++) if (h[b * 4 + 2] < t_min) t_min = h[b * 4 + 2];
  printf("start times (cycles since the first) of blocks 0, 8, 16, ... on their XCC:");
  for (int b = 0; b < 8 * 40; b += 8) printf(" %u", h[b * 4 + 2] - t_min);
  printf("\n");
  return 0;
}
