// A stand-in for librccl.so.1 in a process of its own (tests/fake_rccl_child.py): collectives of this one rank, with what the other ranks would have sent put in by the test, and a device
// allocation that can be made to fail.  Everything is host work on the default stream's results; no kernel is launched here.
#include <cstddef>
#include <dlfcn.h>

extern "C" {
double fake_root_has_muon = 0, fake_others_can = 1; int fake_fail_above = 0;      // the root's third double | the other ranks' least answer | hipMalloc of more bytes than this fails (0: none)
int fake_broadcasts = 0, fake_reduces = 0; size_t fake_last_count = 0; double fake_mine = -1;

static void* hip(const char* name) { static void* lib = dlopen("libamdhip64.so", RTLD_NOW | RTLD_NOLOAD) ? dlopen("libamdhip64.so", RTLD_NOW) : dlopen("/opt/rocm/lib/libamdhip64.so", RTLD_NOW); return lib ? dlsym(lib, name) : nullptr; }
static int copy(void* to, const void* from, size_t n, int kind) { auto f = (int (*)(void*, const void*, size_t, int))hip("hipMemcpy"); return f ? f(to, from, n, kind) : 1; }
int hipMalloc(void** p, size_t n) {
    if (fake_fail_above && n > (size_t)fake_fail_above) { *p = nullptr; return 2; }      // hipErrorOutOfMemory
    auto f = (int (*)(void**, size_t))hip("hipMalloc"); return f ? f(p, n) : 1;
}
int ncclGetUniqueId(void*) { return 0; }
int ncclCommInitRank(void** c, int, char*, int) { static int token; *c = &token; return 0; }
int ncclCommDestroy(void*) { return 0; }
const char* ncclGetErrorString(int) { return "stand-in"; }
int ncclGroupStart() { return 0; }
int ncclGroupEnd() { return 0; }
int ncclBroadcast(const void*, void* recv, size_t count, int type, int, void*, void* stream) {
    ++fake_broadcasts; fake_last_count = count;
    if (type != 8 || count != 3) return 0;                                                // ncclDouble
    auto sync = (int (*)(void*))hip("hipStreamSynchronize"); if (!sync || sync(stream)) return 1;
    return copy((char*)recv + 16, &fake_root_has_muon, 8, 1);
}
int ncclAllReduce(const void* send, void* recv, size_t count, int type, int op, void*, void* stream) {
    ++fake_reduces;
    if (type != 8 || count != 1 || op != 3) return 1;                                     // ncclMin
    auto sync = (int (*)(void*))hip("hipStreamSynchronize"); if (!sync || sync(stream)) return 1;
    if (copy(&fake_mine, send, 8, 2)) return 1;
    const double all = fake_mine < fake_others_can ? fake_mine : fake_others_can;
    return copy(recv, &all, 8, 1);
}
}
