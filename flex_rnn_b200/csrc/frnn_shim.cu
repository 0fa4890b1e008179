// libfrnn_b200.so: NVRTC compile + module load + stream launch behind a C ABI
// (declared in include/frnn.h), plus two small benchmark helper kernels.
//
// libnvrtc and libcuda are opened lazily with dlopen, so the library itself
// loads (and frnn_compile works) on a machine without a GPU or driver.
#include <cuda.h>
#include <cuda_runtime.h>
#include <dlfcn.h>
#include <nvrtc.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/frnn.h"

namespace {

thread_local std::string g_err;

int vfail(int code, const char* fmt, va_list ap) {
    char buf[1024];
    vsnprintf(buf, sizeof buf, fmt, ap);
    g_err = buf;
    return code;
}

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vfail(code, fmt, ap);
    va_end(ap);
    return code;
}

// ---- NVRTC, resolved at first use ------------------------------------------
struct Nvrtc {
    void* lib = nullptr;
    nvrtcResult (*CreateProgram)(nvrtcProgram*, const char*, const char*, int, const char* const*, const char* const*);
    nvrtcResult (*CompileProgram)(nvrtcProgram, int, const char* const*);
    nvrtcResult (*GetProgramLogSize)(nvrtcProgram, size_t*);
    nvrtcResult (*GetProgramLog)(nvrtcProgram, char*);
    nvrtcResult (*GetCUBINSize)(nvrtcProgram, size_t*);
    nvrtcResult (*GetCUBIN)(nvrtcProgram, char*);
    nvrtcResult (*DestroyProgram)(nvrtcProgram*);
    const char* (*GetErrorString)(nvrtcResult);
    nvrtcResult (*Version)(int*, int*);
    std::string why;
};

Nvrtc* nvrtc() {
    static Nvrtc n;
    static std::once_flag once;
    std::call_once(once, [] {
        std::vector<std::string> names;
        if (const char* e = getenv("FRNN_NVRTC_LIB")) names.push_back(e);
        names.push_back("libnvrtc.so.12");
        names.push_back("/usr/local/cuda/lib64/libnvrtc.so.12");
        names.push_back("libnvrtc.so");
        for (auto& nm : names) {
            n.lib = dlopen(nm.c_str(), RTLD_NOW | RTLD_LOCAL);
            if (n.lib) break;
            n.why = dlerror() ? dlerror() : "dlopen failed";
        }
        if (!n.lib) return;
        bool ok = true;
        auto sym = [&](const char* s) {
            void* p = dlsym(n.lib, s);
            if (!p) { ok = false; n.why = std::string("missing symbol ") + s; }
            return p;
        };
        *(void**)&n.CreateProgram = sym("nvrtcCreateProgram");
        *(void**)&n.CompileProgram = sym("nvrtcCompileProgram");
        *(void**)&n.GetProgramLogSize = sym("nvrtcGetProgramLogSize");
        *(void**)&n.GetProgramLog = sym("nvrtcGetProgramLog");
        *(void**)&n.GetCUBINSize = sym("nvrtcGetCUBINSize");
        *(void**)&n.GetCUBIN = sym("nvrtcGetCUBIN");
        *(void**)&n.DestroyProgram = sym("nvrtcDestroyProgram");
        *(void**)&n.GetErrorString = sym("nvrtcGetErrorString");
        *(void**)&n.Version = sym("nvrtcVersion");
        if (!ok) { dlclose(n.lib); n.lib = nullptr; }
    });
    return n.lib ? &n : nullptr;
}

// ---- CUDA driver, resolved at first use --------------------------------------
struct Driver {
    void* lib = nullptr;
    CUresult (*Init)(unsigned);
    CUresult (*CtxGetCurrent)(CUcontext*);
    CUresult (*ModuleLoadData)(CUmodule*, const void*);
    CUresult (*ModuleUnload)(CUmodule);
    CUresult (*ModuleGetFunction)(CUfunction*, CUmodule, const char*);
    CUresult (*FuncSetAttribute)(CUfunction, CUfunction_attribute, int);
    CUresult (*FuncGetAttribute)(int*, CUfunction_attribute, CUfunction);
    CUresult (*LaunchKernel)(CUfunction, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned,
                             CUstream, void**, void**);
    CUresult (*GetErrorString)(CUresult, const char**);
    CUresult (*TensorMapEncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                     const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                     CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    std::string why;
};

Driver* driver() {
    static Driver d;
    static std::once_flag once;
    std::call_once(once, [] {
        d.lib = dlopen("libcuda.so.1", RTLD_NOW | RTLD_LOCAL);
        if (!d.lib) { d.why = dlerror() ? dlerror() : "dlopen libcuda.so.1 failed"; return; }
        bool ok = true;
        auto sym = [&](const char* s) {
            void* p = dlsym(d.lib, s);
            if (!p) { ok = false; d.why = std::string("missing symbol ") + s; }
            return p;
        };
        *(void**)&d.Init = sym("cuInit");
        *(void**)&d.CtxGetCurrent = sym("cuCtxGetCurrent");
        *(void**)&d.ModuleLoadData = sym("cuModuleLoadData");
        *(void**)&d.ModuleUnload = sym("cuModuleUnload");
        *(void**)&d.ModuleGetFunction = sym("cuModuleGetFunction");
        *(void**)&d.FuncSetAttribute = sym("cuFuncSetAttribute");
        *(void**)&d.FuncGetAttribute = sym("cuFuncGetAttribute");
        *(void**)&d.LaunchKernel = sym("cuLaunchKernel");
        *(void**)&d.GetErrorString = sym("cuGetErrorString");
        *(void**)&d.TensorMapEncodeTiled = sym("cuTensorMapEncodeTiled");
        if (!ok) { dlclose(d.lib); d.lib = nullptr; return; }
        d.Init(0);
    });
    return d.lib ? &d : nullptr;
}

const char* cu_str(Driver* d, CUresult r) {
    const char* s = nullptr;
    if (d->GetErrorString(r, &s) != CUDA_SUCCESS || !s) s = "unknown CUDA driver error";
    return s;
}

}  // namespace

// The same for the library's other files (frnn_lm.cuh).
int frnn_fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vfail(code, fmt, ap);
    va_end(ap);
    return code;
}

struct frnn_module {
    CUmodule mod = nullptr;
    std::vector<CUfunction> fn;
};

extern "C" {

int frnn_abi_version(void) { return 2; }

int frnn_nvrtc_version(int* major, int* minor) {
    if (!major || !minor) return fail(FRNN_E_ARG, "frnn_nvrtc_version: bad argument");
    Nvrtc* n = nvrtc();
    if (!n) return fail(FRNN_E_NVRTC, "NVRTC is not available (libnvrtc.so.12 could not be loaded)");
    nvrtcResult r = n->Version(major, minor);
    if (r != NVRTC_SUCCESS) return fail(FRNN_E_NVRTC, "nvrtcVersion: %s", n->GetErrorString(r));
    return FRNN_OK;
}

const char* frnn_last_error(void) { return g_err.c_str(); }

void frnn_free(void* p) { free(p); }

int frnn_compile(const char* src, const char* const* opts, int nopts, void** cubin, size_t* cubin_size,
                 char* log, size_t log_cap) {
    if (log && log_cap) log[0] = 0;
    if (!src || !cubin || !cubin_size || nopts < 0 || (nopts && !opts)) return fail(FRNN_E_ARG, "frnn_compile: bad argument");
    Nvrtc* n = nvrtc();
    if (!n) return fail(FRNN_E_NVRTC, "NVRTC is not available: %s", nvrtc() ? "" : "libnvrtc.so.12 could not be loaded");
    nvrtcProgram prog;
    nvrtcResult r = n->CreateProgram(&prog, src, "frnn_step.cu", 0, nullptr, nullptr);
    if (r != NVRTC_SUCCESS) return fail(FRNN_E_NVRTC, "nvrtcCreateProgram: %s", n->GetErrorString(r));
    std::vector<const char*> o = {"--gpu-architecture=sm_100a", "-std=c++17", "-lineinfo", "--ptxas-options=-v"};
    for (int i = 0; i < nopts; i++) o.push_back(opts[i]);
    r = n->CompileProgram(prog, (int)o.size(), o.data());
    size_t ls = 0;
    if (n->GetProgramLogSize(prog, &ls) == NVRTC_SUCCESS && ls > 1) {
        std::string l(ls, 0);
        n->GetProgramLog(prog, &l[0]);
        if (log && log_cap) {
            size_t c = l.size() < log_cap - 1 ? l.size() : log_cap - 1;
            memcpy(log, l.data(), c);
            log[c] = 0;
        }
        if (r != NVRTC_SUCCESS) {
            n->DestroyProgram(&prog);
            return fail(FRNN_E_NVRTC, "NVRTC compilation failed: %s\n%.700s", n->GetErrorString(r), l.c_str());
        }
    }
    if (r != NVRTC_SUCCESS) {
        n->DestroyProgram(&prog);
        return fail(FRNN_E_NVRTC, "NVRTC compilation failed: %s", n->GetErrorString(r));
    }
    size_t sz = 0;
    r = n->GetCUBINSize(prog, &sz);
    if (r != NVRTC_SUCCESS || sz == 0) {
        n->DestroyProgram(&prog);
        return fail(FRNN_E_NVRTC, "nvrtcGetCUBINSize: %s", n->GetErrorString(r));
    }
    char* buf = (char*)malloc(sz);
    if (!buf) { n->DestroyProgram(&prog); return fail(FRNN_E_ARG, "out of host memory"); }
    r = n->GetCUBIN(prog, buf);
    n->DestroyProgram(&prog);
    if (r != NVRTC_SUCCESS) { free(buf); return fail(FRNN_E_NVRTC, "nvrtcGetCUBIN: %s", n->GetErrorString(r)); }
    *cubin = buf;
    *cubin_size = sz;
    return FRNN_OK;
}

int frnn_module_load(const void* cubin, size_t cubin_size, const char* const* kernel_names,
                     const unsigned* smem_bytes, int nkernels, frnn_module_t* out) {
    if (!cubin || !cubin_size || !kernel_names || nkernels <= 0 || !out) return fail(FRNN_E_ARG, "frnn_module_load: bad argument");
    Driver* d = driver();
    if (!d) return fail(FRNN_E_DRIVER, "CUDA driver is not available (libcuda.so.1)");
    // make sure the runtime's primary context of the current device is current
    cudaError_t ce = cudaFree(0);
    if (ce != cudaSuccess) return fail(FRNN_E_DRIVER, "no usable CUDA device: %s", cudaGetErrorString(ce));
    CUcontext ctx = nullptr;
    d->CtxGetCurrent(&ctx);
    if (!ctx) return fail(FRNN_E_DRIVER, "no current CUDA context");
    frnn_module* m = new frnn_module();
    CUresult r = d->ModuleLoadData(&m->mod, cubin);
    if (r != CUDA_SUCCESS) { delete m; return fail(FRNN_E_DRIVER, "cuModuleLoadData: %s", cu_str(d, r)); }
    for (int i = 0; i < nkernels; i++) {
        CUfunction f;
        r = d->ModuleGetFunction(&f, m->mod, kernel_names[i]);
        if (r != CUDA_SUCCESS) {
            d->ModuleUnload(m->mod);
            delete m;
            return fail(FRNN_E_DRIVER, "kernel '%s' not found: %s", kernel_names[i], cu_str(d, r));
        }
        if (smem_bytes && smem_bytes[i] > 48 * 1024) {
            r = d->FuncSetAttribute(f, CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES, (int)smem_bytes[i]);
            if (r != CUDA_SUCCESS) {
                d->ModuleUnload(m->mod);
                delete m;
                return fail(FRNN_E_LAUNCH, "kernel '%s' needs %u bytes of shared memory: %s", kernel_names[i],
                            smem_bytes[i], cu_str(d, r));
            }
        }
        m->fn.push_back(f);
    }
    *out = m;
    return FRNN_OK;
}

int frnn_module_unload(frnn_module_t m) {
    if (!m) return FRNN_OK;
    Driver* d = driver();
    if (d && m->mod) d->ModuleUnload(m->mod);
    delete m;
    return FRNN_OK;
}

int frnn_launch(frnn_module_t m, int kernel, const unsigned grid[3], const unsigned block[3], unsigned smem_bytes,
                void* stream, void* const* args, int nargs) {
    if (!m || kernel < 0 || kernel >= (int)m->fn.size() || !grid || !block || (nargs && !args))
        return fail(FRNN_E_ARG, "frnn_launch: bad argument");
    Driver* d = driver();
    if (!d) return fail(FRNN_E_DRIVER, "CUDA driver is not available");
    if (!grid[0] || !grid[1] || !grid[2] || !block[0] || block[0] * block[1] * block[2] > 1024)
        return fail(FRNN_E_ARG, "frnn_launch: empty grid or oversized block");
    CUresult r = d->LaunchKernel(m->fn[kernel], grid[0], grid[1], grid[2], block[0], block[1], block[2], smem_bytes,
                                 (CUstream)stream, (void**)args, nullptr);
    if (r != CUDA_SUCCESS) return fail(FRNN_E_LAUNCH, "cuLaunchKernel: %s", cu_str(d, r));
    return FRNN_OK;
}

int frnn_tensor_map_encode(void* out_map, const void* base, unsigned elt_bytes, unsigned rank,
                           const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box) {
    if (!out_map || !base || rank < 1 || rank > 5 || !dims || !box || (rank > 1 && !strides_bytes))
        return fail(FRNN_E_ARG, "frnn_tensor_map_encode: bad argument");
    if (((uintptr_t)out_map & 63) || ((uintptr_t)base & 15))
        return fail(FRNN_E_ARG, "frnn_tensor_map_encode: the map must be 64-byte and the tensor 16-byte aligned");
    Driver* d = driver();
    if (!d) return fail(FRNN_E_DRIVER, "CUDA driver is not available");
    CUtensorMapDataType dt;
    switch (elt_bytes) {
        case 1: dt = CU_TENSOR_MAP_DATA_TYPE_UINT8; break;
        case 2: dt = CU_TENSOR_MAP_DATA_TYPE_UINT16; break;
        case 4: dt = CU_TENSOR_MAP_DATA_TYPE_UINT32; break;
        case 8: dt = CU_TENSOR_MAP_DATA_TYPE_UINT64; break;
        default: return fail(FRNN_E_ARG, "frnn_tensor_map_encode: element size %u", elt_bytes);
    }
    cuuint64_t gd[5], gs[5];
    cuuint32_t bx[5], es[5];
    for (unsigned i = 0; i < rank; i++) { gd[i] = dims[i]; bx[i] = box[i]; es[i] = 1; }
    for (unsigned i = 0; i + 1 < rank; i++) gs[i] = strides_bytes[i];
    CUresult r = d->TensorMapEncodeTiled((CUtensorMap*)out_map, dt, rank, (void*)base, gd, gs, bx, es,
                                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FRNN_E_DRIVER, "cuTensorMapEncodeTiled: %s", cu_str(d, r));
    return FRNN_OK;
}

int frnn_kernel_attrs(frnn_module_t m, int kernel, int* regs, int* static_smem, int* local_bytes) {
    if (!m || kernel < 0 || kernel >= (int)m->fn.size()) return fail(FRNN_E_ARG, "frnn_kernel_attrs: bad argument");
    Driver* d = driver();
    if (!d) return fail(FRNN_E_DRIVER, "CUDA driver is not available");
    if (regs) d->FuncGetAttribute(regs, CU_FUNC_ATTRIBUTE_NUM_REGS, m->fn[kernel]);
    if (static_smem) d->FuncGetAttribute(static_smem, CU_FUNC_ATTRIBUTE_SHARED_SIZE_BYTES, m->fn[kernel]);
    if (local_bytes) d->FuncGetAttribute(local_bytes, CU_FUNC_ATTRIBUTE_LOCAL_SIZE_BYTES, m->fn[kernel]);
    return FRNN_OK;
}

}  // extern "C"

// ---- kernel error word ---------------------------------------------------------

namespace {
const char* kernel_code_text(int code) {
    switch (code) {
        case 1: return "a staged-input copy did not arrive within the wait limit";
        case 2: return "a checkpoint copy did not arrive within the wait limit";
        case 96: return "a token is outside the vocabulary";
        default: return "unknown code";
    }
}
}  // namespace

extern "C" {

int frnn_status_post(int* err_word_dev, int* host_word, void* stream) {
    if (!err_word_dev || !host_word) return fail(FRNN_E_ARG, "frnn_status_post: bad argument");
    cudaError_t e = cudaMemcpyAsync(host_word, err_word_dev, sizeof(int), cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (e != cudaSuccess) return fail(FRNN_E_DRIVER, "frnn_status_post: %s", cudaGetErrorString(e));
    return FRNN_OK;
}

int frnn_status_check(int* host_word, int* err_word_dev, void* stream) {
    if (!host_word) return fail(FRNN_E_ARG, "frnn_status_check: bad argument");
    const int code = *(volatile int*)host_word;
    if (!code) return FRNN_OK;
    *(volatile int*)host_word = 0;
    if (err_word_dev) cudaMemsetAsync(err_word_dev, 0, sizeof(int), (cudaStream_t)stream);   // the word is sticky: clear it
    return fail(FRNN_E_KERNEL, "a kernel reported error %d through its error word (%s); its outputs are not valid",
                code, kernel_code_text(code));
}

int frnn_status(int* err_word_dev, void* stream) {
    if (!err_word_dev) return fail(FRNN_E_ARG, "frnn_status: bad argument");
    int code = 0;
    cudaError_t e = cudaMemcpyAsync(&code, err_word_dev, sizeof(int), cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
    if (e != cudaSuccess) return fail(FRNN_E_DRIVER, "frnn_status: %s", cudaGetErrorString(e));
    if (!code) return FRNN_OK;
    cudaMemsetAsync(err_word_dev, 0, sizeof(int), (cudaStream_t)stream);
    return fail(FRNN_E_KERNEL, "a kernel reported error %d through its error word (%s); its outputs are not valid",
                code, kernel_code_text(code));
}

}  // extern "C"

// ---- launch with the kernel's scratch buffers in library-owned static memory ----

#define FRNN_STATIC_SCRATCH_BYTES (32u << 20)
// Scratch for frnn_launch_static_scratch.  Lives in every CUDA context that loads
// this library until the process exits; shared by all calls on that device.
static __device__ __align__(256) unsigned char frnn_static_scratch[FRNN_STATIC_SCRATCH_BYTES];

namespace {
std::mutex g_scratch_mu;
void* g_scratch_base[64] = {nullptr};   // device address of frnn_static_scratch, per device ordinal
}

extern "C" {

size_t frnn_static_scratch_capacity(void) { return (size_t)FRNN_STATIC_SCRATCH_BYTES; }

int frnn_launch_static_scratch(frnn_module_t m, int kernel, const unsigned grid[3], const unsigned block[3],
                               unsigned smem_bytes, void* stream, void* const* args, int nargs,
                               const int* scratch_arg, const size_t* scratch_bytes, int nscratch) {
    enum { MAX_ARGS = 64 };
    if (!m || !args || nargs <= 0 || nargs > MAX_ARGS || nscratch <= 0 || nscratch > nargs || !scratch_arg || !scratch_bytes)
        return fail(FRNN_E_ARG,
                    "frnn_launch_static_scratch: bad argument (at most %d kernel parameters, and no more scratch "
                    "parameters than kernel parameters)", (int)MAX_ARGS);
    // everything that can be refused is refused before the array is looked up or anything is launched
    // carve 256-byte aligned slices out of the static array; refuse what does not fit
    size_t off[MAX_ARGS];
    bool taken[MAX_ARGS] = {false};
    size_t total = 0;
    for (int i = 0; i < nscratch; i++) {
        if (scratch_arg[i] < 0 || scratch_arg[i] >= nargs)
            return fail(FRNN_E_ARG, "frnn_launch_static_scratch: scratch parameter index %d out of range", scratch_arg[i]);
        if (taken[scratch_arg[i]])
            return fail(FRNN_E_ARG, "frnn_launch_static_scratch: scratch parameter index %d is listed twice", scratch_arg[i]);
        taken[scratch_arg[i]] = true;
        off[i] = total;
        if (scratch_bytes[i] > (size_t)FRNN_STATIC_SCRATCH_BYTES)
            total = (size_t)FRNN_STATIC_SCRATCH_BYTES + 1;
        else
            total += (scratch_bytes[i] + 255) / 256 * 256;
        if (total > (size_t)FRNN_STATIC_SCRATCH_BYTES)
            return fail(FRNN_E_ARG,
                        "frnn_launch_static_scratch: the kernel needs more scratch than the library's static "
                        "buffer holds (capacity %zu bytes); use frnn_launch with caller-allocated scratch",
                        (size_t)FRNN_STATIC_SCRATCH_BYTES);
    }
    if (kernel < 0 || kernel >= (int)m->fn.size() || !grid || !block)
        return fail(FRNN_E_ARG, "frnn_launch_static_scratch: bad kernel index, grid or block");
    if (!grid[0] || !grid[1] || !grid[2] || !block[0] || block[0] * block[1] * block[2] > 1024)
        return fail(FRNN_E_ARG, "frnn_launch_static_scratch: empty grid or oversized block");
    // one-time set-up per device: the host-side name of a __device__ array is not a device
    // address; ask the runtime for the address in the current device's context
    int dev = -1;
    cudaError_t ce = cudaGetDevice(&dev);
    if (ce != cudaSuccess || dev < 0 || dev >= 64)
        return fail(FRNN_E_DRIVER, "frnn_launch_static_scratch: no current CUDA device: %s", cudaGetErrorString(ce));
    void* base = nullptr;
    {
        std::lock_guard<std::mutex> lock(g_scratch_mu);
        if (!g_scratch_base[dev]) {
            void* p = nullptr;
            ce = cudaGetSymbolAddress(&p, frnn_static_scratch);
            if (ce != cudaSuccess || !p)
                return fail(FRNN_E_DRIVER, "frnn_launch_static_scratch: cudaGetSymbolAddress failed: %s",
                            cudaGetErrorString(ce));
            g_scratch_base[dev] = p;
        }
        base = g_scratch_base[dev];
    }
    // parameter list with the scratch pointers substituted (stack storage only)
    void* slot[MAX_ARGS];
    void* argv[MAX_ARGS];
    for (int i = 0; i < nargs; i++) argv[i] = args[i];
    for (int i = 0; i < nscratch; i++) {
        slot[i] = (unsigned char*)base + off[i];
        argv[scratch_arg[i]] = &slot[i];
    }
    return frnn_launch(m, kernel, grid, block, smem_bytes, stream, argv, nargs);
}

}  // extern "C"

// ---- benchmark helpers --------------------------------------------------------

__global__ void frnn_flush_kernel(uint4* p, size_t n16, unsigned v) {
    size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    size_t stride = (size_t)gridDim.x * blockDim.x;
    uint4 x = make_uint4(v, v, v, v);
    for (; i < n16; i += stride) p[i] = x;
}

// 16 independent FMA chains per thread, all in registers: the FP32 pipe is the
// only resource in use.
__global__ void __launch_bounds__(256) frnn_fma_probe_kernel(float* sink, int iters) {
    float a[16];
#pragma unroll
    for (int i = 0; i < 16; i++) a[i] = 1.0f + 1e-3f * (threadIdx.x + i);
    const float m = 0.9999f, c = 1e-4f;
    for (int it = 0; it < iters; it++) {
#pragma unroll
        for (int u = 0; u < 8; u++) {
#pragma unroll
            for (int i = 0; i < 16; i++) a[i] = fmaf(a[i], m, c);
        }
    }
    float s = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) s += a[i];
    if (s == 12345.678f) sink[0] = s;  // never true; keeps the chains alive
}

// ---- what the FP32 pipe delivers for the recurrent kernels' kinds of FMA -------------------------
// Register-only loops (no memory, no shuffles).  The register file feeds two 32-bit operands per thread and
// clock, an FMA reads three: FMAs whose three operands are all distinct registers run at about two thirds of
// the rate of FMAs that keep one operand from the previous instruction.  The scan kernels' FMAs are of the first
// kind wherever the compiler's instruction order does not happen to repeat an operand.

// kind 0 / 1: scalar FFMA, three distinct register operands / one operand shared by all instructions
template <int SHARED> __global__ void __launch_bounds__(256) frnn_mix_ffma_kernel(float* sink, const float* in, int iters) {
    float a[32], b[32], d[32];
#pragma unroll
    for (int i = 0; i < 32; i++) { a[i] = in[threadIdx.x % 7 + i]; b[i] = in[threadIdx.x % 5 + i + 3]; d[i] = in[i]; }
    for (int it = 0; it < iters; it++) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
#pragma unroll
            for (int i = 0; i < 32; i++) d[i] = fmaf(SHARED ? a[0] : a[i], b[i], d[i]);
        }
    }
    float s = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) s += d[i];
    if (s == 12345.678f) sink[0] = s;
}

// kind 2 / 3: packed FFMA2 (two fp32 lanes per instruction), three distinct register pairs / one pair shared
template <int SHARED> __global__ void __launch_bounds__(256) frnn_mix_ffma2_kernel(float* sink, const float* in, int iters) {
    float2 a[32], b[32], d[32];
#pragma unroll
    for (int i = 0; i < 32; i++) {
        a[i] = make_float2(in[threadIdx.x % 7 + i], in[threadIdx.x % 7 + i + 1]);
        b[i] = make_float2(in[threadIdx.x % 5 + i + 3], in[threadIdx.x % 5 + i + 4]);
        d[i] = make_float2(in[i], in[i + 1]);
    }
    for (int it = 0; it < iters; it++) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
#pragma unroll
            for (int i = 0; i < 32; i++) d[i] = __ffma2_rn(SHARED ? a[0] : a[i], b[i], d[i]);
        }
    }
    float s = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) s += d[i].x + d[i].y;
    if (s == 12345.678f) sink[0] = s;
}

#define FRNN_P(v, i) make_float2((v)[i], (v)[(i) + 1])
#define FRNN_BB(x) make_float2((x), (x))
#define FRNN_ST(v, i, e) { const float2 t_ = (e); (v)[i] = t_.x; (v)[(i) + 1] = t_.y; }
// kind 4: the seven FMAs per state element of the Delta Rule backward step on an 8x8 register tile of the state (s)
// and of its gradient (d), packed, one pass per graph node as the code generator emits them:
// A = dS' + dy q^T; dq += S'^T dy; w = -(A bk); e += A^T u; dS = A + w q^T; S = S' - u bk^T; f += S^T w
__global__ void __launch_bounds__(256, 1) frnn_mix_delta_bw_kernel(float* sink, const float* in, int iters) {
    float s[64], d[64], a[8], b[8], q[8], y[8];
#pragma unroll
    for (int i = 0; i < 64; i++) { s[i] = in[threadIdx.x + i]; d[i] = in[threadIdx.x + i + 7]; }
#pragma unroll
    for (int i = 0; i < 8; i++) { a[i] = in[i + threadIdx.x % 3]; b[i] = in[64 + i + threadIdx.x % 5]; q[i] = in[99 + i]; y[i] = in[33 + i]; }
    for (int it = 0; it < iters; it++) {
        float t[64], n[8], p0[8], p1[8], p2[8];
#pragma unroll
        for (int c = 0; c < 8; c++) { p0[c] = 0; p1[c] = 0; p2[c] = 0; }
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
            for (int c = 0; c < 8; c += 2) FRNN_ST(t, r * 8 + c, __ffma2_rn(FRNN_BB(y[r]), FRNN_P(q, c), FRNN_P(d, r * 8 + c)));
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
            for (int c = 0; c < 8; c += 2) FRNN_ST(p0, c, __ffma2_rn(FRNN_BB(y[r]), FRNN_P(s, r * 8 + c), FRNN_P(p0, c)));
#pragma unroll
        for (int r = 0; r < 8; r++) {
            float2 acc = FRNN_BB(0.f);
#pragma unroll
            for (int c = 0; c < 8; c += 2) acc = __ffma2_rn(FRNN_P(t, r * 8 + c), FRNN_P(a, c), acc);
            n[r] = -(acc.x + acc.y);
        }
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
            for (int c = 0; c < 8; c += 2) FRNN_ST(p1, c, __ffma2_rn(FRNN_P(t, r * 8 + c), FRNN_BB(b[r]), FRNN_P(p1, c)));
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
            for (int c = 0; c < 8; c += 2) FRNN_ST(d, r * 8 + c, __ffma2_rn(FRNN_BB(n[r]), FRNN_P(q, c), FRNN_P(t, r * 8 + c)));
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
            for (int c = 0; c < 8; c += 2) FRNN_ST(s, r * 8 + c, __ffma2_rn(FRNN_P(a, c), FRNN_BB(-b[r]), FRNN_P(s, r * 8 + c)));
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
            for (int c = 0; c < 8; c += 2) FRNN_ST(p2, c, __ffma2_rn(FRNN_BB(n[r]), FRNN_P(s, r * 8 + c), FRNN_P(p2, c)));
#pragma unroll
        for (int c = 0; c < 8; c++) q[c] += (p0[c] + p1[c] + p2[c]) * 1e-9f;
#pragma unroll
        for (int r = 0; r < 8; r++) y[r] += n[r] * 1e-9f;
    }
    float acc = 0;
#pragma unroll
    for (int i = 0; i < 64; i++) acc += s[i] + d[i];
#pragma unroll
    for (int i = 0; i < 8; i++) acc += q[i] + y[i];
    if (acc == 12345.678f) sink[0] = acc;
}

// kind 5: the three FMAs per state element of the Delta Rule forward step on a 4x32 register tile, scalar:
// sk = S k; S += (v - sk) bk^T; y = S q   (two accumulators per row sum)
__global__ void __launch_bounds__(256, 1) frnn_mix_delta_fw_kernel(float* sink, const float* in, int iters) {
    float S[128], q[32], kk[32], bk[32], v[4];
#pragma unroll
    for (int i = 0; i < 128; i++) S[i] = in[threadIdx.x + i];
#pragma unroll
    for (int i = 0; i < 32; i++) { q[i] = in[i + threadIdx.x % 3]; kk[i] = in[64 + i + threadIdx.x % 5]; bk[i] = in[99 + i]; }
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = in[33 + i];
    for (int it = 0; it < iters; it++) {
        float a1[8], a2[8], u[4], y[4];
#pragma unroll
        for (int i = 0; i < 8; i++) { a1[i] = 0.f; a2[i] = 0.f; }
#pragma unroll
        for (int c = 0; c < 32; c++)
#pragma unroll
            for (int r = 0; r < 4; r++) a1[r * 2 + c % 2] = fmaf(S[r * 32 + c], kk[c], a1[r * 2 + c % 2]);
#pragma unroll
        for (int r = 0; r < 4; r++) u[r] = v[r] - (a1[2 * r] + a1[2 * r + 1]);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int c = 0; c < 32; c++) S[r * 32 + c] = fmaf(bk[c], u[r], S[r * 32 + c]);
#pragma unroll
        for (int c = 0; c < 32; c++)
#pragma unroll
            for (int r = 0; r < 4; r++) a2[r * 2 + c % 2] = fmaf(S[r * 32 + c], q[c], a2[r * 2 + c % 2]);
#pragma unroll
        for (int r = 0; r < 4; r++) { y[r] = a2[2 * r] + a2[2 * r + 1]; v[r] += y[r] * 1e-9f; }
    }
    float acc = 0;
#pragma unroll
    for (int i = 0; i < 128; i++) acc += S[i];
#pragma unroll
    for (int i = 0; i < 4; i++) acc += v[i];
    if (acc == 12345.678f) sink[0] = acc;
}

extern "C" {

int frnn_fp32_mix_probe(int kind, float* sink, const float* in, int iters, void* stream, double* flops) {
    if (!sink || !in || iters <= 0 || kind < 0 || kind > 5) return fail(FRNN_E_ARG, "frnn_fp32_mix_probe: bad argument");
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (sms <= 0) return fail(FRNN_E_DRIVER, "no CUDA device");
    cudaStream_t st = (cudaStream_t)stream;
    double per_thread = 0;
    switch (kind) {
        case 0: frnn_mix_ffma_kernel<0><<<sms, 256, 0, st>>>(sink, in, iters); per_thread = 2.0 * 32 * 4; break;
        case 1: frnn_mix_ffma_kernel<1><<<sms, 256, 0, st>>>(sink, in, iters); per_thread = 2.0 * 32 * 4; break;
        case 2: frnn_mix_ffma2_kernel<0><<<sms, 256, 0, st>>>(sink, in, iters); per_thread = 2.0 * 64 * 4; break;
        case 3: frnn_mix_ffma2_kernel<1><<<sms, 256, 0, st>>>(sink, in, iters); per_thread = 2.0 * 64 * 4; break;
        case 4: frnn_mix_delta_bw_kernel<<<sms, 256, 0, st>>>(sink, in, iters); per_thread = 2.0 * 64 * 7; break;
        default: frnn_mix_delta_fw_kernel<<<sms, 256, 0, st>>>(sink, in, iters); per_thread = 2.0 * 128 * 3; break;
    }
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(FRNN_E_LAUNCH, "frnn_fp32_mix_probe: %s", cudaGetErrorString(e));
    if (flops) *flops = per_thread * (double)iters * sms * 256;
    return FRNN_OK;
}

int frnn_l2_flush(void* buf, size_t bytes, void* stream) {
    if (!buf || bytes < 16) return fail(FRNN_E_ARG, "frnn_l2_flush: bad argument");
    static std::atomic<unsigned> pattern{0};
    frnn_flush_kernel<<<1184, 256, 0, (cudaStream_t)stream>>>((uint4*)buf, bytes / 16, ++pattern);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(FRNN_E_LAUNCH, "frnn_l2_flush: %s", cudaGetErrorString(e));
    return FRNN_OK;
}

int frnn_fp32_peak_probe(float* sink, int iters, void* stream, double* flops) {
    if (!sink || iters <= 0) return fail(FRNN_E_ARG, "frnn_fp32_peak_probe: bad argument");
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (sms <= 0) return fail(FRNN_E_DRIVER, "no CUDA device");
    const int blocks = sms * 8, threads = 256;
    frnn_fma_probe_kernel<<<blocks, threads, 0, (cudaStream_t)stream>>>(sink, iters);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(FRNN_E_LAUNCH, "frnn_fp32_peak_probe: %s", cudaGetErrorString(e));
    if (flops) *flops = 2.0 * 16 * 8 * (double)iters * blocks * threads;
    return FRNN_OK;
}

}  // extern "C"
