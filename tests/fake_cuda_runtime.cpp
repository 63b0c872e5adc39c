// A CUDA runtime without a GPU, for tests of the library's host code: memory is a range of addresses that nothing is stored at, kernels are
// noted and not run.  What it keeps: every allocation, every launch with its stream and (for kernels that a test watches) its arguments,
// and for streams, events and synchronisation a clock per stream, from which follows which launch comes before which.
// Calls that the real runtime refuses, or that are undefined there, are counted as misuse: a destroyed stream's handle, an
// allocation or a wait of the host while a stream is being captured.
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cstring>
#include <map>
#include <string>
#include <vector>

namespace {

using Clock = std::map<unsigned long long, long>;  // stream id -> operations of it that have come before

struct Stream {
    unsigned long long id;
    bool alive, capturing;
    Clock clock;
};
struct Launch {
    std::string name;
    unsigned long long stream;
    bool captured;
    Clock before;  // its own place included
    std::vector<std::vector<unsigned char>> args;
};
struct Watch { std::string part; std::vector<int> sizes; };
struct Config { dim3 grid, block; size_t smem; cudaStream_t stream; };

std::map<uintptr_t, size_t> alive, freed;
std::map<cudaStream_t, Stream> streams;
std::map<const void*, std::string> kernels;
std::vector<Launch> launches;
std::vector<Watch> watches;
std::vector<Config> configs;
std::vector<std::string> misuse;
Clock host, gone;  // gone: what destroyed streams had been given
uintptr_t next_address = 0x100000000000ull;
unsigned long long next_id = 2;
uintptr_t next_handle = 0x5000;
size_t bytes_alive = 0;
cudaStreamCaptureMode mode = cudaStreamCaptureModeGlobal;  // of the calling thread
constexpr size_t MEMORY = (size_t)180 << 30;

void merge(Clock& to, const Clock& from) {
    for (auto& e : from)
        if (to[e.first] < e.second) to[e.first] = e.second;
}
bool capturing() {
    for (auto& s : streams)
        if (s.second.alive && s.second.capturing) return true;
    return false;
}
Stream* find(cudaStream_t s, const char* call) {
    if (!s && !streams.count(s)) streams[s] = Stream{1, true, false, {}};
    auto at = streams.find(s);
    if (at == streams.end() || !at->second.alive) {
        misuse.push_back(std::string(call) + " on a stream that does not exist");
        return nullptr;
    }
    return &at->second;
}
cudaError_t while_capturing(const char* call) {
    misuse.push_back(std::string(call) + " while a stream is being captured");
    return cudaErrorStreamCaptureUnsupported;
}
cudaError_t launch(const void* func, void** args, cudaStream_t stream) {
    Stream* s = find(stream, "a launch");
    if (!s) return cudaErrorContextIsDestroyed;
    Launch l;
    l.name = kernels.count(func) ? kernels[func] : "?";
    l.stream = s->id;
    l.captured = s->capturing;
    merge(s->clock, host);
    ++s->clock[s->id];
    l.before = s->clock;
    for (auto& w : watches)
        if (l.name.find(w.part) != std::string::npos)
            for (size_t i = 0; i < w.sizes.size(); ++i) {
                const unsigned char* p = (const unsigned char*)args[i];
                l.args.emplace_back(p, p + w.sizes[i]);
            }
    launches.push_back(l);
    return cudaSuccess;
}
CUresult encode(CUtensorMap* map, ...) {
    memset(map, 0, sizeof(*map));
    return CUDA_SUCCESS;
}

}  // namespace

extern "C" {

// ---- what the tests ask ----
void fake_watch(const char* part, const int* sizes, int n) { watches.push_back(Watch{part, std::vector<int>(sizes, sizes + n)}); }
int fake_launches() { return (int)launches.size(); }
void fake_forget_launches() { launches.clear(); }
const char* fake_launch_name(int i) { return launches[i].name.c_str(); }
int fake_launch_captured(int i) { return launches[i].captured; }
int fake_launch_args(int i) { return (int)launches[i].args.size(); }
void fake_launch_arg(int i, int k, void* out) { memcpy(out, launches[i].args[k].data(), launches[i].args[k].size()); }
int fake_comes_before(int i, int j) {
    const Launch &a = launches[i], &b = launches[j];
    auto at = b.before.find(a.stream);
    return at != b.before.end() && at->second >= a.before.at(a.stream);
}
size_t fake_room_behind(uintptr_t p) {  // bytes from p to the end of its allocation, 0 outside
    auto at = alive.upper_bound(p);
    if (at == alive.begin()) return 0;
    --at;
    return p < at->first + at->second ? at->first + at->second - p : 0;
}
size_t fake_bytes_alive() { return bytes_alive; }
int fake_misuse() { return (int)misuse.size(); }
const char* fake_misuse_text(int i) { return misuse[i].c_str(); }
uintptr_t fake_stream_create(uintptr_t handle) {  // 0: a new handle
    if (!handle) handle = next_handle += 16;
    else if (streams.count((cudaStream_t)handle)) merge(gone, streams[(cudaStream_t)handle].clock);
    streams[(cudaStream_t)handle] = Stream{next_id++, true, false, {}};
    return handle;
}
void fake_stream_destroy(uintptr_t handle) { streams[(cudaStream_t)handle].alive = false; }
void fake_capture(uintptr_t handle, int on) { find((cudaStream_t)handle, "capture")->capturing = on != 0; }

// ---- memory ----
cudaError_t cudaMalloc(void** p, size_t n) {
    if (capturing() && mode != cudaStreamCaptureModeRelaxed) return while_capturing("cudaMalloc");
    if (bytes_alive + n > MEMORY) return cudaErrorMemoryAllocation;
    *p = (void*)next_address;
    alive[next_address] = n;
    bytes_alive += n;
    next_address += (n + (4u << 20)) & ~(uintptr_t)0xFFFFF;
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
    if (!p) return cudaSuccess;
    if (capturing()) return while_capturing("cudaFree");
    auto at = alive.find((uintptr_t)p);
    if (at == alive.end()) {
        misuse.push_back("cudaFree of what is not allocated");
        return cudaErrorInvalidValue;
    }
    bytes_alive -= at->second;
    freed[at->first] = at->second;
    alive.erase(at);
    for (auto& s : streams)
        if (s.second.alive) merge(host, s.second.clock);
    return cudaSuccess;
}
cudaError_t cudaFreeHost(void*) { return cudaSuccess; }
cudaError_t cudaMemset(void*, int, size_t) { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t s) { return find(s, "cudaMemsetAsync") ? cudaSuccess : cudaErrorContextIsDestroyed; }
cudaError_t cudaMemcpy(void* dst, const void*, size_t n, cudaMemcpyKind kind) {
    if (kind == cudaMemcpyDeviceToHost) memset(dst, 0, n);
    return cudaSuccess;
}
cudaError_t cudaMemcpyAsync(void*, const void*, size_t, cudaMemcpyKind, cudaStream_t s) { return find(s, "cudaMemcpyAsync") ? cudaSuccess : cudaErrorContextIsDestroyed; }
cudaError_t cudaIpcGetMemHandle(cudaIpcMemHandle_t*, void*) { return cudaErrorNotSupported; }
cudaError_t cudaIpcOpenMemHandle(void**, cudaIpcMemHandle_t, unsigned) { return cudaErrorNotSupported; }
cudaError_t cudaIpcCloseMemHandle(void*) { return cudaErrorNotSupported; }
cudaError_t cudaGetSymbolAddress(void**, const void*) { return cudaErrorNotSupported; }

// ---- device ----
cudaError_t cudaGetDeviceCount(int* n) { *n = 1; return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) {
    memset(p, 0, sizeof(*p));
    p->major = 10;
    p->multiProcessorCount = 148;
    p->sharedMemPerBlockOptin = 232448;
    return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 1965000; return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() {
    if (capturing()) return while_capturing("cudaDeviceSynchronize");
    for (auto& s : streams) merge(host, s.second.clock);  // a destroyed stream's work too
    merge(host, gone);
    return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long, cudaDriverEntryPointQueryResult* q) {
    *fn = (void*)encode;
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "error of the runtime without a GPU"; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }

// ---- streams and events ----
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) {
    const cudaStreamCaptureMode before = mode;
    mode = *m;
    *m = before;
    return cudaSuccess;
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { *s = (cudaStream_t)fake_stream_create(0); return cudaSuccess; }
cudaError_t cudaStreamDestroy(cudaStream_t s) {
    if (!find(s, "cudaStreamDestroy")) return cudaErrorContextIsDestroyed;
    streams[s].alive = false;
    return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t s) {
    Stream* at = find(s, "cudaStreamSynchronize");
    if (!at) return cudaErrorContextIsDestroyed;
    if (at->capturing) return while_capturing("cudaStreamSynchronize");
    merge(host, at->clock);
    return cudaSuccess;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t s, cudaStreamCaptureStatus* status) {
    Stream* at = find(s, "cudaStreamIsCapturing");
    if (!at) return cudaErrorContextIsDestroyed;
    *status = at->capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
    return cudaSuccess;
}
cudaError_t cudaStreamGetId(cudaStream_t s, unsigned long long* id) {
    Stream* at = find(s, "cudaStreamGetId");
    if (!at) return cudaErrorContextIsDestroyed;
    *id = at->id;
    return cudaSuccess;
}
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t e, unsigned) {
    Stream* at = find(s, "cudaStreamWaitEvent");
    if (!at) return cudaErrorContextIsDestroyed;
    merge(at->clock, *(Clock*)e);
    return cudaSuccess;
}
cudaError_t cudaEventCreate(cudaEvent_t* e) { *e = (cudaEvent_t) new Clock; return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return cudaEventCreate(e); }
cudaError_t cudaEventDestroy(cudaEvent_t e) { delete (Clock*)e; return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) {
    Stream* at = find(s, "cudaEventRecord");
    if (!at) return cudaErrorContextIsDestroyed;
    *(Clock*)e = at->clock;
    return cudaSuccess;
}
cudaError_t cudaEventElapsedTime_v2(float* ms, cudaEvent_t, cudaEvent_t) { *ms = 0; return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float* ms, cudaEvent_t, cudaEvent_t) { *ms = 0; return cudaSuccess; }

// ---- kernels ----
cudaError_t cudaLaunchKernel(const void* func, dim3, dim3, void** args, size_t, cudaStream_t s) { return launch(func, args, s); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* func, void** args) { return launch(func, args, c->stream); }
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t smem, struct CUstream_st* stream) {
    configs.push_back(Config{grid, block, smem, stream});
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* grid, dim3* block, size_t* smem, void* stream) {
    const Config c = configs.back();
    configs.pop_back();
    *grid = c.grid;
    *block = c.block;
    *smem = c.smem;
    *(cudaStream_t*)stream = c.stream;
    return cudaSuccess;
}
void** __cudaRegisterFatBinary(void*) { static void* none; return &none; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char* host_fun, char*, const char* name, int, uint3*, uint3*, dim3*, dim3*, int*) { kernels[host_fun] = name; }
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}

}  // extern "C"
