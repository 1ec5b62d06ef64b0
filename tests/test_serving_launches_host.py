"""What the host code of the serving operators asks the CUDA runtime for, on the CPU: their objects linked with a runtime that launches nothing
and refuses what the real one would. Calls by two threads at once, sizes of grids and shared memory."""
import re
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

# The limits are those of compute capability 10.0: 48 KB of dynamic shared memory unless more was asked for, 227 KB in all; grids of up to 2^31 - 1, 65535, 65535.
# What a real call may take long for takes 40 ms here, so that a second thread always comes in between.
RUNTIME = r"""
#include <cuda.h>
#include <cuda_runtime_api.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <mutex>
#include <thread>
#include <vector>
#include "cacheir_b200_serving.h"

static std::mutex lock;
static std::map<const void*, int> allowed;
static std::vector<dim3> grids;
static int lowered = 0, asked = 0;
static std::atomic<int> waits{0};
static void wait_ms(int ms) { std::this_thread::sleep_for(std::chrono::milliseconds(ms)); }

extern "C" {
void** __cudaRegisterFatBinary(void*) { static void* handle = nullptr; return &handle; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
unsigned __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return 1; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaGetDevice(int* device) { *device = 0; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaMemcpyFromSymbol(void* to, const void*, size_t n, size_t, cudaMemcpyKind) { for (size_t i = 0; i < n; ++i) static_cast<char*>(to)[i] = 0; return cudaSuccess; }
cudaError_t cudaMemcpyToSymbol(const void*, const void*, size_t, size_t, cudaMemcpyKind) { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* kernel, cudaFuncAttribute what, int value) {
  {
    std::lock_guard<std::mutex> hold(lock);
    if (what != cudaFuncAttributeMaxDynamicSharedMemorySize || value < 0 || value > 227 * 1024) return cudaErrorInvalidValue;
    if (allowed.count(kernel) && value < allowed[kernel]) ++lowered;
    allowed[kernel] = value;
    ++asked;
  }
  if (waits) wait_ms(40);
  return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* cfg, const void* kernel, void**) {
  std::lock_guard<std::mutex> hold(lock);
  const size_t most = allowed.count(kernel) && allowed[kernel] > 48 * 1024 ? allowed[kernel] : 48 * 1024;
  const dim3 g = cfg->gridDim, b = cfg->blockDim;
  if (cfg->dynamicSmemBytes > most || g.x == 0 || g.y == 0 || g.z == 0 || g.x > 0x7fffffffu || g.y > 65535 || g.z > 65535 || b.x * b.y * b.z > 1024)
    return cudaErrorInvalidValue;
  grids.push_back(g);
  return cudaSuccess;
}
static CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t rank, void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                       const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
  if (reinterpret_cast<uintptr_t>(base) % 16) return CUDA_ERROR_INVALID_VALUE;
  for (cuuint32_t i = 0; i < rank; ++i)
    if (dims[i] == 0 || dims[i] > 1ull << 32 || box[i] == 0 || box[i] > 256 || (i > 0 && (strides[i - 1] % 16 || strides[i - 1] >= 1ull << 40))) return CUDA_ERROR_INVALID_VALUE;
  return CUDA_SUCCESS;
}
cudaError_t cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long, cudaDriverEntryPointQueryResult* found) {
  if (waits) wait_ms(40);
  *fn = reinterpret_cast<void*>(&encode);
  *found = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
}

// (addresses that nothing looks at)
static int attention(int batch, int heads, int kv_heads, int dim, int dtype, int groups, int page_size = 16) {
  void* some = reinterpret_cast<void*>(size_t{1} << 32);
  cacheir_b200_prefix_args a{};
  a.q = a.k_cache = a.v_cache = some;
  a.out = a.workspace = some;
  a.page_table = a.seq_lens = a.group_rows = a.prefix_table = a.prefix_lens = static_cast<int32_t*>(some);
  a.workspace_bytes = cacheir_b200_shared_prefix_workspace_bytes(batch, heads, dim);
  a.q_stride = a.out_stride = static_cast<long long>(heads) * dim;
  a.batch = batch;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.page_size = page_size;
  a.num_slots = 64;
  a.max_pages = a.prefix_pages = 4;
  a.groups = groups;
  a.dtype = dtype;
  return cacheir_b200_shared_prefix_attention(&a, nullptr);
}
template <typename A, typename B>
static void beside(A first, B second) {
  waits = 1;
  std::thread one(first), two([&] { wait_ms(10); second(); });
  one.join();
  two.join();
  waits = 0;
}
"""


def _run(tmp_path, main):
    from cacheir_b200 import build

    build.build(groups=("serving",))
    include = Path(build.find_nvcc()).resolve().parents[1] / "include"
    (tmp_path / "calls.cpp").write_text(RUNTIME + "int main() {\n" + main + "\n}\n")
    objects = [str(build.BUILD_DIR / (src.stem + ".o")) for src in build.group_sources("serving")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(include), "-I", str(build.INCLUDE), "calls.cpp", *objects, "-o", "calls"], cwd=tmp_path,
                   check=True)
    done = subprocess.run([str(tmp_path / "calls")], capture_output=True, text=True, check=True, timeout=60)
    return [[int(v) for v in line.split()] for line in done.stdout.splitlines()]


def test_first_calls_of_two_threads_find_the_encoder_of_copies(tmp_path):
    """What makes the descriptors of copies is looked up by the first call. One that comes in meanwhile waits for it instead of finding nothing."""
    [codes] = _run(tmp_path, """
  int a = 1, b = 1;
  beside([&] { a = attention(4, 8, 2, 128, CACHEIR_B200_F16, 1); }, [&] { b = attention(4, 8, 2, 64, CACHEIR_B200_BF16, 1); });
  std::printf("%d %d\\n", a, b);""")
    assert codes == [0, 0]


def test_every_lookup_of_the_encoder_is_made_once_for_all_threads():
    for source in sorted((ROOT / "cacheir_b200" / "csrc").glob("*.cu*")):
        for call in re.finditer(r"cudaGetDriverEntryPoint\(", text := source.read_text()):
            assert re.search(r"static const EncodeTiledFn fn = \[\] \{[^}]*$", text[: call.start()]), source.name


def test_shared_memory_of_a_kernel_never_shrinks(tmp_path):
    """Head sizes of the general attention kernels need 36 to 148 KB. What a kernel may have holds for all threads: a call with a smaller head must
    not take from another what that has just asked for. It is asked for once per element type."""
    two, after = _run(tmp_path, """
  int a = 1, b = 1;
  beside([&] { a = attention(4, 8, 2, 512, CACHEIR_B200_F32, 1); }, [&] { b = attention(4, 8, 2, 96, CACHEIR_B200_F32, 1); });
  std::printf("%d %d\\n", a, b);
  asked = 0;
  for (int dtype : {CACHEIR_B200_F32, CACHEIR_B200_F16, CACHEIR_B200_BF16})
    for (int dim : {512, 80, 512, 33})
      if (attention(4, 8, 2, dim, dtype, 1)) return 1;
  std::printf("%d %d\\n", lowered, asked);""")
    assert two == [0, 0]
    assert after == [0, 2]


def test_general_attention_takes_any_number_of_rows_that_the_entry_takes(tmp_path):
    """Tiles of the general kernels go where a grid is widest. Rows, heads per key/value head, groups: what counted 65536 tiles and more was refused."""
    [codes] = _run(tmp_path, """
  const int codes[] = {attention(65535, 8, 8, 80, CACHEIR_B200_F32, 65535), attention(4096, 64, 1, 80, CACHEIR_B200_BF16, 1), attention(65535, 64, 1, 64, CACHEIR_B200_F32, 0),
                       attention(65535, 8, 1, 64, CACHEIR_B200_F16, 3, 8), attention(65536, 8, 8, 80, CACHEIR_B200_F32, 1)};
  for (int code : codes) std::printf("%d ", code);""")
    assert codes == [0, 0, 0, 0, -5]
