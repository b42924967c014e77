// split_ws.cu — see split_ws.h.
#include "split_ws.h"

#include <mutex>

namespace tsn {

namespace {

constexpr size_t WORKSPACE = SPLIT_GROUPS * 4 + SPLIT_BYTES;

// Host calls that touch no stream of the program, so that they also work while one of them is being captured.
struct Uncaptured {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    Uncaptured() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~Uncaptured() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
cudaError_t zero(void * p, size_t bytes) {   // and waits for it
    Uncaptured u;
    cudaStream_t s = nullptr;
    cudaError_t e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, bytes, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (s) cudaStreamDestroy(s);
    return e;
}
cudaError_t allocate(void ** p, size_t bytes) {
    Uncaptured u;
    return cudaMalloc(p, bytes);
}
int failed(const char * name, cudaError_t e) {
    cudaGetLastError();
    return fail(e == cudaErrorMemoryAllocation ? TSN_ERR_OOM : TSN_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
}

// The device's workspace, ordered after the last call that used it. Streams are told apart by their id, which no other
// stream of the process ever has: a handle may stand for one stream per thread, or be given out again.
int workspace(DeviceCtx & c, const char * name, unsigned long long stream) {
    cudaError_t e = cudaSuccess;
    if (!c.split_ws) {
        void * p = nullptr;
        e = allocate(&p, WORKSPACE);
        if (e == cudaSuccess) e = zero(p, SPLIT_GROUPS * 4);
        if (e == cudaSuccess && !c.split_ev) e = cudaEventCreateWithFlags(&c.split_ev, cudaEventDisableTiming);
        if (e != cudaSuccess) { cudaFree(p); return failed(name, e); }
        c.split_ws = p;
    }
    if (c.split_used && c.split_stream != stream) e = cudaStreamWaitEvent(c.stream, c.split_ev, 0);
    return e == cudaSuccess ? TSN_OK : failed(name, e);
}

// Workspaces of captured calls. One belongs to its call's graph, so that replays need no order among themselves or with other
// calls; when the graph and its executables are gone it lies here until another capture, or the device's end, takes it.
struct Block {
    void * p;
    size_t bytes;
    int ordinal;
    Block * next;
};
std::mutex g_idle_mu;
Block * g_idle = nullptr;

void CUDART_CB make_idle(void * block) {   // no CUDA calls in here
    std::lock_guard<std::mutex> lk(g_idle_mu);
    Block * b = (Block *) block;
    b->next = g_idle;
    g_idle = b;
}

int graph_workspace(const DeviceCtx & c, const char * name, cudaGraph_t graph, size_t bytes, void ** out) {
    size_t size = (size_t) 1 << 18;   // powers of two, so that they fit the calls of later captures
    while (size < bytes) size *= 2;
    Block * b = nullptr;
    {
        std::lock_guard<std::mutex> lk(g_idle_mu);
        for (Block ** at = &g_idle; *at; at = &(*at)->next)
            if ((*at)->ordinal == c.ordinal && (*at)->bytes == size) {
                b = *at;
                *at = b->next;
                break;
            }
    }
    if (!b) {
        b = new Block{nullptr, size, c.ordinal, nullptr};
        const cudaError_t e = allocate(&b->p, size);
        if (e != cudaSuccess) { delete b; return failed(name, e); }
    }
    cudaUserObject_t object = nullptr;
    cudaError_t e = zero(b->p, size);
    if (e == cudaSuccess) e = cudaUserObjectCreate(&object, b, make_idle, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) {
        make_idle(b);
        return failed(name, e);
    }
    e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) {
        cudaUserObjectRelease(object, 1);
        return failed(name, e);
    }
    *out = b->p;
    return TSN_OK;
}

} // namespace

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
        cudaDriverEntryPointQueryResult q{};
        void * fn = nullptr;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return (PFN_cuTensorMapEncodeTiled_v12000) fn;
    }();
    return enc;
}

void release_split(int ordinal) {
    Block * gone = nullptr;
    {
        std::lock_guard<std::mutex> lk(g_idle_mu);
        for (Block ** at = &g_idle; *at;) {
            Block * b = *at;
            if (b->ordinal != ordinal) { at = &b->next; continue; }
            *at = b->next;
            b->next = gone;
            gone = b;
        }
    }
    while (gone) {   // without the lock: freeing may wait for a thread of the driver's that is in make_idle
        Block * b = gone;
        gone = b->next;
        cudaFree(b->p);
        delete b;
    }
}

int split_begin(DeviceCtx & c, const char * name, size_t groups, size_t bytes, SplitUse & u) {
    cudaGraph_t graph = nullptr;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamGetCaptureInfo(c.stream, &capture, nullptr, &graph, nullptr, nullptr);
    if (e == cudaSuccess && capture == cudaStreamCaptureStatusInvalidated) e = cudaErrorStreamCaptureInvalidated;
    if (e == cudaSuccess && capture == cudaStreamCaptureStatusNone) e = cudaStreamGetId(c.stream, &u.stream);
    if (e != cudaSuccess) return failed(name, e);
    u.captured = capture != cudaStreamCaptureStatusNone;
    size_t counters = SPLIT_GROUPS * 4;
    void * ws = nullptr;
    int rc;
    if (!u.captured) {
        rc = workspace(c, name, u.stream);
        ws = c.split_ws;
    } else {
        counters = (groups * 4 + 255) & ~(size_t) 255;
        rc = graph_workspace(c, name, graph, counters + bytes, &ws);
    }
    if (rc) return rc;
    u.count = (unsigned int *) ws;
    u.part = (float *) ((char *) ws + counters);
    return TSN_OK;
}

cudaError_t split_end(DeviceCtx & c, const SplitUse & u) {
    if (u.captured) return cudaSuccess;
    const cudaError_t e = cudaEventRecord(c.split_ev, c.stream);
    c.split_used = true;
    c.split_stream = u.stream;
    return e;
}

} // namespace tsn
