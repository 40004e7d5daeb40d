// Stands in for the CUDA runtime and for the kernels behind deepj_b200/csrc/runtime.cu, so that what the interpreter checks, counts and hands to its
// launchers can be tested without a GPU: buffers are host memory, copies and additions are done, every other launch is noted down.
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <vector>

#include <cuda_runtime.h>

#include "kernels.h"

namespace {
struct Note { int kind, a, b, c; };               // kind: an op code
std::vector<Note> notes;
void note(int kind, int a = 0, int b = 0, int c = 0) { dj::g_launches++; notes.push_back({kind, a, b, c}); }
}  // namespace

extern "C" {
int standin_notes(int* out, int most) {           // what was launched since the last call, four numbers each
    const int n = (int)notes.size();
    for (int i = 0; i < n && i < most; i++) std::memcpy(out + 4 * i, &notes[i], sizeof(Note));
    notes.clear();
    return n;
}

void** __cudaRegisterFatBinary(void*) { static void* handle; return &handle; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
char __cudaInitModule(void**) { return 1; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) { std::memset((void*)p, 0, sizeof *p); p->major = 10; p->multiProcessorCount = 148; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t e) { return e == cudaErrorMemoryAllocation ? "out of memory" : "error"; }
cudaError_t cudaMalloc(void** p, size_t n) { *p = n > (size_t)1 << 33 ? nullptr : std::malloc(n); return *p ? cudaSuccess : cudaErrorMemoryAllocation; }
cudaError_t cudaFree(void* p) { std::free(p); return cudaSuccess; }
cudaError_t cudaMallocHost(void** p, size_t n) { *p = std::malloc(n); return cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { std::free(p); return cudaSuccess; }
cudaError_t cudaMemset(void* p, int v, size_t n) { std::memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t) { std::memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { std::memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) { std::memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemcpy2DAsync(void* d, size_t dp, const void* s, size_t sp, size_t w, size_t h, cudaMemcpyKind, cudaStream_t) {
    for (size_t i = 0; i < h; i++) std::memcpy((char*)d + i * dp, (const char*)s + i * sp, w);
    return cudaSuccess;
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { *s = nullptr; return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamBeginCapture(cudaStream_t, cudaStreamCaptureMode) { return cudaSuccess; }
cudaError_t cudaStreamEndCapture(cudaStream_t, cudaGraph_t* g) { *g = nullptr; return cudaErrorUnknown; }      // the interpreter then launches one by one
cudaError_t cudaGraphDestroy(cudaGraph_t) { return cudaSuccess; }
cudaError_t cudaGraphExecDestroy(cudaGraphExec_t) { return cudaSuccess; }
cudaError_t cudaGraphInstantiate(cudaGraphExec_t*, cudaGraph_t, unsigned long long) { return cudaErrorUnknown; }
cudaError_t cudaGraphLaunch(cudaGraphExec_t, cudaStream_t) { return cudaErrorUnknown; }
cudaError_t cudaEventCreate(cudaEvent_t* e) { *e = nullptr; return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float* ms, cudaEvent_t, cudaEvent_t) { *ms = 0.0f; return cudaSuccess; }
cudaError_t cudaGetDriverEntryPoint(const char*, void** f, unsigned long long, cudaDriverEntryPointQueryResult* r) { *f = nullptr; *r = cudaDriverEntryPointSymbolNotFound; return cudaSuccess; }
}  // extern "C"

namespace dj {
// what the launchers do where there is nothing to do: they launch nothing
void launch_copy(const float* src, float* dst, long long n, cudaStream_t) { if (n > 0) { std::memmove(dst, src, (size_t)n * 4); note(70); } }
void launch_add_scalar_inplace(float* b, float v, int n, cudaStream_t) { if (n > 0) { for (int i = 0; i < n; i++) b[i] += v; note(69); } }
void launch_binary(int op, const float* a, const float* b, float* out, int n, cudaStream_t) { if (n > 0) { for (int i = 0; i < n; i++) out[i] = a[i] + b[i]; note(op); } }
void launch_embed_gather(const float*, const float*, float*, int rows, int, int, cudaStream_t) { if (rows > 0) note(64, rows); }
void launch_argmax_rows(const float*, float* out, int rows, int, int*, int*, cudaStream_t) { for (int i = 0; i < rows; i++) out[i] = 0.0f; if (rows > 0) note(68, rows); }
size_t sample_topk_ws_floats(int, int, int) { return 0; }
void launch_sample_topk(const float*, const float*, float* out, int rows, int, int, float, float*, cudaStream_t) { for (int i = 0; i < rows; i++) out[i] = 0.0f; note(74, rows); }
void launch_synth_fill(float* p, unsigned long long, unsigned long long, float, long long, long long n, cudaStream_t) { std::memset(p, 0, (size_t)n * 4); }
void launch_q8_quantize(const float*, int, int, int, int8_t*, float*, int, int, cudaStream_t) { g_launches++; }
void launch_q8_linear(const Q8LinearArgs& a, cudaStream_t) { note(65, a.M); }
size_t q8_batch_ws_floats(int, int, bool) { return 0; }
size_t q8_tc_ws_floats(int, int, int, bool) { return 0; }
bool tp_ready() { return false; }

size_t q4_plane_bytes(int B, int G, int maxSeq, int hd) { return (size_t)B * G * ((maxSeq + 31) / 32) * 36 * hd; }
size_t q4_attn_ws_floats(const Q4AttnArgs&) { return 0; }
size_t q4_decode_ws_floats(const Q4AttnArgs&) { return 0; }
size_t q4_evict_ws_floats(const Q4EvictArgs&) { return 0; }
void launch_q4_append(const Q4AttnArgs& a, int T, cudaStream_t) { note(90, a.M, T); }
void launch_q4_attn(const Q4AttnArgs& a, cudaStream_t) { if (a.M > 0 || a.accOut != nullptr) note(88, a.M, a.H, a.G); }
void launch_q4_decode(const Q4AttnArgs& a, cudaStream_t) {
    if (a.accOut != nullptr) a.accOut[0] = a.acc[0] + 1.0f;          // weights are added up
    note(87, a.early, a.H, a.G);
}
void launch_q4_load(const Q4LoadArgs& a, cudaStream_t) { if (a.T > 0) note(91, a.T); }
void launch_q4_evict(const Q4EvictArgs& a, cudaStream_t) {
    for (int b = 0; b < a.B; b++) {
        a.lenOut[b] = std::fmin(std::fmax(a.len[b], 0.0f), (float)a.budget);
        note(89, b, (int)a.len[b], a.budget);
    }
}
}  // namespace dj
