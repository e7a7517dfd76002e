"""What the sources of the tensor-core kernels must keep to, read from the sources: breaking it stops a GPU instead of failing a test there.

Tensor memory is given out by an instruction that waits for as long as it takes, so no block may wait for tensor memory that is held by
one that waits for it."""
import os
import re

import pytest

from fms_b200.kernels.build import CSRC


def without_comments(text):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def kernels():
    """(file, name, body) of every kernel that takes tensor memory."""
    found = []
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = without_comments(f.read())
        for part in re.split(r"\b__global__\b", text)[1:]:
            part = part[: part.index("\n}")]  # a kernel ends at the first brace in the first column
            if "tmem_alloc" in part:
                kernel = re.search(r"(\w+_kernel)\s*\(", part).group(1)
                found.append(pytest.param(part, id=f"{name}:{kernel}"))
    return found


KERNELS = kernels()


def test_every_file_with_tensor_memory_is_looked_at():
    files = {p.id.split(":")[0] for p in KERNELS}
    assert files >= {"attention_tc.cuh", "attention_f32_tc.cuh", "gemm_bf16_mid.cu", "gemm_bf16_tc.cu", "gemm_e4m3.cu", "gemm_f32_tc.cu", "gemm_int4.cu"}
    assert sum("tmem_alloc_pair" in p.values[0] for p in KERNELS) == 3


@pytest.mark.parametrize("body", KERNELS)
def test_a_pair_takes_its_tensor_memory_when_both_blocks_run(body):
    """The two blocks of a pair take theirs together: either needs the other to be there, which a cluster's barrier says."""
    if "tmem_alloc_pair" in body:
        at = body.index("tmem_alloc_pair(")
        assert "cluster_sync_all();" in body[:at]
        assert body[at:].index("cluster_sync_all();") < body[at:].index("elect_one()")  # and nothing is issued before both have theirs


@pytest.mark.parametrize("body", KERNELS)
def test_the_next_kernel_is_let_in_when_a_block_has_its_tensor_memory(body):
    """A block of the next kernel takes tensor memory and waits for this kernel: had it come in earlier, it could hold what a block of
    this kernel still waits for."""
    if "pdl_launch_dependents" in body:
        taken = body.rindex("tmem_alloc")
        assert body.index("pdl_launch_dependents") > taken + body[taken:].index("__syncthreads();")


def test_a_warp_comes_together_before_an_instruction_of_all_of_it():
    """tcgen05 instructions and cluster barriers that are .aligned are reached by all lanes at once: behind a loop that some lanes go
    around early the compiler need not see to that."""
    seen = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = without_comments(f.read())
        for found in re.finditer(r"(tcgen05|barrier\.cluster)[\w.:]*\.aligned", text):
            function = text[text.rindex("__forceinline__", 0, found.start()): found.start()]
            assert "__syncwarp();" in function, (name, found.group(0))
            seen += 1
    assert seen >= 18
