"""What the host code of the operators of drafted tokens asks the CUDA runtime for, on the CPU: their objects linked with a runtime that launches nothing and
refuses what the real one would. Sizes of grids and shared memory, first calls of two threads."""
import subprocess
from pathlib import Path

from test_serving_launches_host import RUNTIME

CALLS = r"""
#include "cacheir_b200_drafts.h"
static void* const some = reinterpret_cast<void*>(size_t{1} << 32);
static int32_t* const ints = static_cast<int32_t*>(some);
static int tree(int rows, int sequences, int heads, int kv_heads, int dim, int dtype, int page_size = 16, int max_pages = 4) {
  cacheir_b200_tree_args a{};
  a.q = a.k_cache = a.v_cache = some;
  a.out = a.workspace = some;
  a.page_table = a.seq_lens = a.cu_rows = ints;
  a.workspace_bytes = cacheir_b200_tree_attention_workspace_bytes(rows, heads, dim);
  a.q_stride = a.out_stride = static_cast<long long>(heads) * dim;
  a.rows = rows;
  a.sequences = sequences;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.page_size = page_size;
  a.num_slots = 64;
  a.max_pages = max_pages;
  a.dtype = dtype;
  return cacheir_b200_tree_attention(&a, nullptr);
}
static int logits(int rows, int vocab, int dtype, int words, int biases, int history) {
  cacheir_b200_logits_args a{};
  a.logits = some;
  a.out = some;
  a.history = history ? ints : nullptr;
  a.history_lens = ints;
  a.history_width = history;
  a.draft_ids = words ? static_cast<int64_t*>(some) : nullptr;
  a.cu_rows = a.visible = ints;
  a.words = words;
  a.bias_ids = ints;
  a.bias_values = static_cast<float*>(some);
  a.biases = biases;
  a.rows = a.sequences = rows;
  a.vocab = vocab;
  a.dtype = a.out_dtype = dtype;
  return cacheir_b200_adjust_logits(&a, nullptr);
}
static int norm(int rows, int dim, int dtype) {
  cacheir_b200_norm_rotary_args n{};
  cacheir_b200_rotary_args& a = n.rotary;
  a.q = a.k = a.q_out = a.k_out = some;
  a.positions = ints;
  a.turns = static_cast<uint64_t*>(some);
  a.q_stride = a.q_out_stride = 4LL * dim;
  a.k_stride = a.k_out_stride = 2LL * dim;
  a.rows = rows;
  a.heads = 4;
  a.kv_heads = 2;
  a.dim = dim;
  a.rot = dim / 2 * 2;
  a.dtype = dtype;
  a.factor = 1.f;
  return cacheir_b200_norm_rotary_append(&n, nullptr);
}
static int drafts(int rows, int sequences, int pools) {
  cacheir_b200_draft_map_args m{ints, ints, ints, ints, ints, ints, rows, sequences, 32};
  cacheir_b200_accept_args c{static_cast<int64_t*>(some), static_cast<int64_t*>(some), ints, ints, ints, ints, ints, static_cast<int64_t*>(some), ints, rows, sequences, 9};
  std::vector<void*> all(pools, some);
  cacheir_b200_keep_args k{all.data(), ints, ints, ints, ints, pools, rows, sequences, 9, 4, 8, 16, 128, CACHEIR_B200_F16};
  int code = cacheir_b200_map_drafts(&m, nullptr);
  if (code == 0) code = cacheir_b200_accept_drafts(&c, nullptr);
  return code == 0 ? cacheir_b200_keep_accepted(&k, nullptr) : code;
}
"""


def _run(tmp_path, main):
    from cacheir_b200 import build

    build.build(groups=("drafts",))
    build.build(groups=("serving",))
    include = Path(build.find_nvcc()).resolve().parents[1] / "include"
    (tmp_path / "calls.cpp").write_text(RUNTIME + CALLS + "int main() {\n" + main + "\n}\n")
    objects = [str(build.BUILD_DIR / (src.stem + ".o")) for group in ("drafts", "serving") for src in build.group_sources(group)]
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(include), "-I", str(build.INCLUDE), "calls.cpp", *objects, "-o", "calls"], cwd=tmp_path,
                   check=True)
    done = subprocess.run([str(tmp_path / "calls")], capture_output=True, text=True, check=True, timeout=60)
    return [[int(v) for v in line.split()] for line in done.stdout.splitlines()]


def test_grids_and_shared_memory_of_the_largest_and_the_smallest_calls(tmp_path):
    """Calls at the documented limits are launched, those past them refused."""
    codes = _run(tmp_path, """
  std::printf("%d %d %d %d %d %d %d\\n", tree(1, 1, 1, 1, 128, CACHEIR_B200_F16), tree(1 << 24, 65535, 8, 8, 128, CACHEIR_B200_BF16), tree(65535, 65535, 64, 1, 64, CACHEIR_B200_F16),
              tree(1 << 20, 65535, 8, 8, 512, CACHEIR_B200_F32), tree(300, 3, 80, 1, 128, CACHEIR_B200_F16), tree(300, 3, 8, 2, 128, CACHEIR_B200_F16, 8),
              tree(9, 3, 8, 2, 64, CACHEIR_B200_F16, 16, 1 << 26));
  std::printf("%d %d %d %d %d %d\\n", logits(1, 1, CACHEIR_B200_F32, 32, 300, 7), logits(524280, 9, CACHEIR_B200_F16, 32, 1, 1), logits(524281, 9, CACHEIR_B200_F16, 0, 0, 0),
              logits(2, 1 << 28, CACHEIR_B200_BF16, 0, 5, 0), logits(65536, 33, CACHEIR_B200_F32, 1, 0, 0), logits(2, 100, CACHEIR_B200_F16, 0, 0, 1 << 29));
  for (int dtype : {CACHEIR_B200_F32, CACHEIR_B200_F16, CACHEIR_B200_BF16})
    for (int dim : {1024, 512, 256, 128, 64, 96, 33, 2}) std::printf("%d ", norm(dim == 128 ? 1 << 24 : 3, dim, dtype));
  std::printf("\\n%d %d %d\\n", drafts(1, 1, 1), drafts(1 << 24, 65535, 300), drafts(9, 65536, 1));""")
    assert codes == [[0] * 7, [0, 0, -5, 0, 0, -5], [0] * 24, [0, 0, -5]]


def test_first_calls_of_two_threads(tmp_path):
    """Both find the encoder of copy descriptors, and neither takes shared memory from the other."""
    [codes] = _run(tmp_path, """
  int a = 1, b = 1, c = 1, d = 1;
  beside([&] { a = tree(4, 2, 8, 2, 128, CACHEIR_B200_F16); }, [&] { b = tree(4, 2, 8, 2, 64, CACHEIR_B200_BF16); });
  beside([&] { c = tree(4, 2, 8, 2, 512, CACHEIR_B200_F32); }, [&] { d = tree(4, 2, 8, 2, 96, CACHEIR_B200_F32); });
  std::printf("%d %d %d %d %d\\n", a, b, c, d, lowered);""")
    assert codes == [0, 0, 0, 0, 0]
