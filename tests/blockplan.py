"""Which kernels the residual block's calls launch, found on the host: block.c
over stand-ins for the pool, the workspace and the HIP calls, which write down
each launch and run nothing. The GPU tests ask it, too, that a case runs the
kernel it is there for."""
import ctypes as C
import functools
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
MOST = 1000          # launches a call may make here: the next one fails

STANDINS = r"""
#include "%(csrc)s/block.c"
HipbState hipb;
const unsigned char thvm_norm_kernels_co[1], thvm_gemm_kernels_co[1];
static HipbBuf buf;
HipbBuf *pool_get(u32 id) { (void)id; return &buf; }
void *pool_ptr(u32 id) { return (void *)((uintptr_t)id << 44); }
u64 pool_bytes(u32 id) { (void)id; return ~0ull; }
void pool_mark_device_write(u32 id) { (void)id; }
void *pool_block_get(u64 bytes, u64 *cap) { (void)bytes; *cap = bytes; return (void *)4096; }
void pool_block_put(void *p, u64 cap) { (void)p; (void)cap; }
void hipb_operand(u32 id) { (void)id; }
static u64 workspace;
void *scratch_reserve(Scratch *s, u64 bytes) { (void)s; workspace = bytes; return (void *)(1ull << 60); }
void scratch_release(Scratch *s) { (void)s; }
static char *names[KERNELS];
hipError_t hipModuleGetFunction(hipFunction_t *f, hipModule_t m, const char *name) {
    (void)m;
    u32 i = 0;
    while (names[i] && strcmp(names[i], name)) i++;
    if (!names[i]) names[i] = strdup(name);
    *f = (hipFunction_t)names[i];
    return hipSuccess;
}
hipError_t hipModuleLoadData(hipModule_t *m, const void *p) { (void)p; *m = NULL; return hipSuccess; }
hipError_t hipModuleUnload(hipModule_t m) { (void)m; return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
const char *hipGetErrorString(hipError_t e) { (void)e; return ""; }
hipFunction_t rtc_static_fn(const char *name) { (void)name; return NULL; }
typedef struct { char name[48]; u32 gx, gy, gz, bx; u64 first, rows; } Launch;
static Launch launches[%(most)d];
static u32 n;
int hipb_launch(hipFunction_t fn, u32 gx, u32 gy, u32 gz, u32 bx, void **params) {
    if (n == %(most)d) return 0;
    Launch *l = &launches[n++];
    snprintf(l->name, sizeof l->name, "%%s", (const char *)fn);
    l->gx = gx; l->gy = gy; l->gz = gz; l->bx = bx; l->first = l->rows = 0;
    if (!strncmp(l->name, "thvm_ln_", 8)) {
        const LnArgs *a = params[0];
        l->first = a->x; l->rows = a->rows;
    } else if (!strncmp(l->name, "thvm_few", 8) || !strncmp(l->name, "thvm_direct", 11) || !strncmp(l->name, "thvm_gemm", 9)) {
        const GemmArgs *a = params[0];
        l->first = a->A; l->rows = a->M;
    }
    return 1;
}
void plan_begin(u32 n_cu) { hipb.initialized = 1; hipb.n_cu = n_cu; n = 0; workspace = 0; }
u32 plan_launches(Launch **l) { *l = launches; return n; }
"""


class Launch(C.Structure):
    _fields_ = [("name", C.c_char * 48), ("gx", C.c_uint32), ("gy", C.c_uint32), ("gz", C.c_uint32), ("bx", C.c_uint32),
                ("first", C.c_uint64), ("rows", C.c_uint64)]


@functools.cache
def _plans():
    csrc = os.path.join(ROOT, "tinyhvm_amd", "csrc")
    with tempfile.TemporaryDirectory() as d:
        src, so = os.path.join(d, "plan.c"), os.path.join(d, "plan.so")
        with open(src, "w") as f:
            f.write(STANDINS % {"csrc": csrc, "most": MOST})
        subprocess.run(["gcc", "-std=gnu11", "-O1", "-w", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROCM, "include"),
                        "-I" + os.path.join(ROOT, "include"), "-I" + csrc, src, "-lm", "-o", so], check=True)
        L = C.CDLL(so)
    f32, u32 = C.c_float, C.c_uint32
    L.thvm_hip_layer_norm.argtypes = [u32] * 8 + [f32, u32]
    L.thvm_hip_muon_step.argtypes = [C.POINTER(u32)] * 3 + [u32] * 3 + [f32] * 4 + [u32] * 3
    return L


def launches(call, *args, n_cu=256, rc=0):
    """The launches (name, gx, gy, gz, bx, first, rows) of a call, whose
    operands may be any ids but 0; first and rows: address and rows of x."""
    L = _plans()
    L.plan_begin(n_cu)
    assert getattr(L, call)(*args) == rc
    p = C.POINTER(Launch)()
    return [p[i] for i in range(L.plan_launches(C.byref(p)))]


def names(call, *args, **kw):
    return [v.name.decode() for v in launches(call, *args, **kw)]


def linear(m, k, n, dtype):
    """The kernels of a layer's call, in order."""
    return names("thvm_hip_linear", 1, 2, 3, 4, 5, 6, 1, m, k, n, dtype)


def linear_grad(m, k, n, dtype):
    return names("thvm_hip_linear_grad", 1, 2, 3, 4, 5, 6, 7, 1, m, k, n, dtype)


def muon_step(count, rows, cols, dtype):
    ids = [(C.c_uint32 * count)(*range(i * count + 1, (i + 1) * count + 1)) for i in range(3)]
    return names("thvm_hip_muon_step", *ids, count, rows, cols, 0.1, 1.0, 0.0, 0.9, 1, 5, dtype)
