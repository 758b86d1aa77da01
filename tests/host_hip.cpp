// A HIP runtime without a GPU, for tests of what the library's host code asks
// of HIP: loaded with RTLD_GLOBAL ahead of libaotk.so, its functions take the
// place of the runtime's. Memory is host memory, copies happen at once, kernels
// are counted and not run. Streams know whether they are captured and by whom;
// gates hold a call in the middle so that two threads meet there.
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include <chrono>
#include <condition_variable>
#include <mutex>
#include <thread>

namespace {
constexpr int OK = 0, INVALID_VALUE = 1, INVALID_DEVICE = 101, CAPTURE_UNSUPPORTED = 900, CAPTURE_INVALIDATED = 901;

struct Dim3 {
    unsigned x, y, z;
};
struct Stream {
    bool capturing = false, broken = false;
    std::thread::id by;
    int device = 0;
    long queued = 0;  // launches that nothing has waited for
};
struct Gate {
    bool armed = false, reached = false, open = false;
};

std::mutex mu;
std::condition_variable cv;
Gate gates[2];
int devices = 1, captured_on = -1;
long launched = 0, foreign = 0, fail_in = 0;
thread_local int device = 0, last = OK;
thread_local struct {
    Dim3 grid, block;
    size_t lds;
    void *stream;
} config;

int done(int e) {
    if (e != OK) last = e;
    return e;
}

void pass(int g) {
    std::unique_lock<std::mutex> l(mu);
    if (!gates[g].armed) return;
    gates[g].armed = false;
    gates[g].reached = true;
    cv.notify_all();
    cv.wait_for(l, std::chrono::seconds(20), [&] { return gates[g].open; });
}
}  // namespace

extern "C" {

// ------------------------------------------------------------ for the tests
void hh_devices(int n) { devices = n; }
// gate 0: a capture has begun; gate 1: a stream was asked whether it is captured
void hh_arm(int gate) {
    std::lock_guard<std::mutex> l(mu);
    gates[gate] = Gate{true, false, false};
}
int hh_reached(int gate, int ms) {
    std::unique_lock<std::mutex> l(mu);
    return cv.wait_for(l, std::chrono::milliseconds(ms), [&] { return gates[gate].reached; });
}
void hh_open(int gate) {
    std::lock_guard<std::mutex> l(mu);
    gates[gate].open = true;
    gates[gate].armed = false;
    cv.notify_all();
}
long hh_launched() { return launched; }
long hh_foreign() { return foreign; }  // launches that went into another thread's capture
int hh_captured_on() { return captured_on; }  // the device of the stream that was captured last
long hh_queued(void *s) { return ((Stream *)s)->queued; }
void hh_fail_launch(long n) { fail_in = n; }  // the n-th launch from here on fails
void hh_set_last_error(int e) { last = e; }

// ------------------------------------------------------------------ devices
int hipGetDeviceCount(int *n) { *n = devices; return OK; }
int hipGetDevice(int *d) { *d = device; return OK; }
int hipSetDevice(int d) {
    if (d < 0 || d >= devices) return done(INVALID_DEVICE);
    device = d;
    return OK;
}
int hipDeviceGetAttribute(int *v, int, int) { *v = 256; return OK; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *, int, size_t) { *n = 1; return OK; }
int hipFuncSetAttribute(const void *, int, int) { return OK; }
const char *hipGetErrorString(int e) { return e == OK ? "no error" : "an error of the stand-in"; }
int hipGetLastError() {
    const int e = last;
    last = OK;
    return e;
}

// ------------------------------------------------------------------- memory
int hipMalloc(void **p, size_t n) { *p = calloc(1, n); return *p ? OK : done(2); }
int hipFree(void *p) { free(p); return OK; }
int hipHostMalloc(void **p, size_t n, unsigned) { return hipMalloc(p, n); }
int hipHostFree(void *p) { return hipFree(p); }
int hipMemcpy(void *d, const void *s, size_t n, int) { memmove(d, s, n); return OK; }
int hipMemcpyAsync(void *d, const void *s, size_t n, int, void *) { memmove(d, s, n); return OK; }
int hipMemsetAsync(void *d, int v, size_t n, void *) { memset(d, v, n); return OK; }
int hipGetSymbolAddress(void **p, const void *s) { *p = (void *)s; return OK; }

// ------------------------------------------------------------------ streams
int hipStreamCreateWithFlags(void **s, unsigned) {
    Stream *x = new Stream;
    x->device = device;
    *s = x;
    return OK;
}
int hipStreamDestroy(void *s) { delete (Stream *)s; return OK; }
int hipStreamSynchronize(void *p) {
    std::lock_guard<std::mutex> l(mu);
    Stream *s = (Stream *)p;
    if (s->capturing) {
        s->broken = true;
        return done(CAPTURE_UNSUPPORTED);
    }
    s->queued = 0;
    return OK;
}
int hipStreamIsCapturing(void *p, int *status) {
    {
        std::lock_guard<std::mutex> l(mu);
        *status = ((Stream *)p)->capturing;
    }
    pass(1);
    return OK;
}
int hipStreamBeginCapture(void *p, int) {
    {
        std::lock_guard<std::mutex> l(mu);
        Stream *s = (Stream *)p;
        if (s->capturing) return done(CAPTURE_UNSUPPORTED);
        s->capturing = true;
        s->broken = false;
        captured_on = s->device;
        s->by = std::this_thread::get_id();
    }
    pass(0);
    return OK;
}
int hipStreamEndCapture(void *p, void **graph) {
    std::lock_guard<std::mutex> l(mu);
    Stream *s = (Stream *)p;
    s->capturing = false;
    *graph = s->broken ? nullptr : malloc(1);
    return s->broken ? done(CAPTURE_INVALIDATED) : OK;
}
int hipGraphInstantiate(void **exec, void *, void **, char *, size_t) { *exec = malloc(1); return OK; }
int hipGraphLaunch(void *, void *) { return OK; }
int hipGraphDestroy(void *g) { free(g); return OK; }
int hipGraphExecDestroy(void *e) { free(e); return OK; }
int hipEventCreate(void **e) { *e = malloc(1); return OK; }
int hipEventDestroy(void *e) { free(e); return OK; }
int hipEventRecord(void *, void *) { return OK; }
int hipEventSynchronize(void *) { return OK; }
int hipEventElapsedTime(float *ms, void *, void *) { *ms = 1; return OK; }

// ----------------------------------------------------------------- launches
void **__hipRegisterFatBinary(const void *) { static void *h; return &h; }
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, void *, void *, int *) {}
void __hipRegisterVar(void **, void *, char *, const char *, int, size_t, int, int) {}
int __hipPushCallConfiguration(Dim3 grid, Dim3 block, size_t lds, void *s) {
    config = {grid, block, lds, s};
    return OK;
}
int __hipPopCallConfiguration(Dim3 *grid, Dim3 *block, size_t *lds, void **s) {
    *grid = config.grid;
    *block = config.block;
    *lds = config.lds;
    *s = config.stream;
    return OK;
}
int hipLaunchKernel(const void *, Dim3, Dim3, void **, size_t, void *p) {
    std::lock_guard<std::mutex> l(mu);
    if (fail_in && --fail_in == 0) return done(INVALID_VALUE);
    Stream *s = (Stream *)p;
    if (s->capturing) {
        if (s->by != std::this_thread::get_id()) foreign++;
        return OK;
    }
    launched++;
    s->queued++;
    return OK;
}

}  // extern "C"
