/* Loads the model of the working directory (graph.json, params.bin) on the fake device, to which table-activated dense layers and
 * staged copies are added, and prints the tables that the launches were prepared with, "@<layer>=value,value,...".
 *
 * Staged copies: cudaMemcpy() of up to 64 KB from ordinary host memory may return when the bytes are staged; they land later, in
 * order, and streams made with cudaStreamNonBlocking do not wait for them.  Here they land when cudaMemcpy() next has to wait, or
 * when the model is loaded.  (Linked with --wrap=cudaMemcpy.)
 *   lut early|late
 */
#include <cuda_runtime.h>
#include <cstdio>
#include <cstring>
#include <deque>
#include <fstream>
#include <iterator>
#include <string>
#include <vector>
#include "cvm/c_api.h"
#include "cvmk_kernels.h"
#include "fake_device.h"

namespace {
struct Staged { void* to; std::vector<char> bytes; };
std::deque<Staged> staged;
std::vector<cvmk_dense_lut_desc> prepared;

void land() {
  for (; !staged.empty(); staged.pop_front()) memcpy(staged.front().to, staged.front().bytes.data(), staged.front().bytes.size());
}
std::string slurp(const char* path) {
  std::ifstream f(path, std::ios::binary);
  return std::string(std::istreambuf_iterator<char>(f), std::istreambuf_iterator<char>());
}
}  // namespace

extern "C" {
cudaError_t __real_cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind kind);
cudaError_t __wrap_cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind kind) {
  if (kind == cudaMemcpyHostToDevice && n <= 65536) {
    staged.push_back({d, std::vector<char>((const char*)s, (const char*)s + n)});
    return cudaSuccess;
  }
  land();
  return __real_cudaMemcpy(d, s, n, kind);
}
int cvmk_dense_lut_supported(const cvmk_dense_lut_desc*) { return 1; }
int cvmk_dense_lut_prepare(const cvmk_dense_lut_desc* d, cvmk_dense_lut_plan* plan) {
  memset(plan, 0, sizeof(*plan));
  plan->d = *d;
  prepared.push_back(*d);
  return CVMK_OK;
}
int cvmk_dense_lut_launch(const cvmk_dense_lut_plan*, cvmk_stream_t) { return CVMK_OK; }
}

int main(int argc, char** argv) {
  if (argc < 2) return 2;
  const std::string graph = slurp("graph.json"), params = slurp("params.bin");
  fake::late = std::string(argv[1]) == "late";
  void* net = nullptr;
  if (CVMAPILoadModel(graph.data(), (int)graph.size(), params.data(), (int)params.size(), &net, 1, 0) != 0) return 3;
  land();
  for (size_t i = 0; i < prepared.size(); ++i) {
    const cvmk_dense_lut_desc& d = prepared[i];
    printf("@%zu=", i);
    for (int j = 0; j < d.table_len; ++j) printf("%s%d", j ? "," : "", d.table_dtype == CVMK_I8 ? ((const int8_t*)d.table)[j] : ((const int32_t*)d.table)[j]);
    printf("\n");
  }
  CVMAPIFreeModel(net);
  return 0;
}
