"""What the paged-cache kernels' order rests on, read from their source: no GPU needed.  They are resident while the
kernels before them still write (programmatic dependent launch), so a slip here shows on a GPU only by chance."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "anedvd_b200", "csrc")
FILES = ["paged.cu", "paged.cuh", "paged_attn.cu", "paged_attn_tc.cu", "paged_mass.cu", "paged_tc.cuh"]


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", FILES)
def test_no_read_takes_the_read_only_path(name):
    """ld.global.nc is for data that no one writes while the kernel lives; that of an earlier grid in flight is not."""
    found = re.findall(r"__ldg\b|\bld\.global\.nc\b|__restrict__", source(name))
    assert not found


def kernels(name):
    """(name, body) of each __global__ function of a file."""
    s = source(name)
    for m in re.finditer(r"__global__.*?(\w+)\s*\((?:[^()]|\([^()]*\))*\)\s*\{", re.sub(r"__launch_bounds__\([^)]*\)", lambda m: " " * len(m[0]), s), re.S):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(s[i], 0)
            i += 1
        yield m[1], s[m.end():i - 1]


def test_every_kernel_is_found():
    assert {k for f in FILES for k, _ in kernels(f)} >= {
        "rope_append_kernel", "evict_select_kernel", "evict_move_kernel", "attn_few_kernel", "attn_merge_kernel",
        "attn_many_kernel", "mass_kernel"}


@pytest.mark.parametrize("name", FILES)
def test_kernels_wait_before_they_read(name):
    """Each kernel waits for what the stream holds before it, in every thread, before it reads lengths, tables or
    tensors: another grid's having waited does not make them visible to this one."""
    for kernel, body in kernels(name):
        head, wait, _ = body.partition("griddep_wait();")
        assert wait, kernel
        assert head.count("{") == head.count("}") and not re.search(r"\b(if|for|while|return)\b[^;]*$", head), kernel
        reads = re.findall(r"\.(?:len|tokens|page|sequence_of|range)\(|\bFewSeq\b|\*\s*reinterpret_cast<const|"
                           r"\b(?:q_start|kv_len|pages|positions|kept|mass|lse)\s*\[|\[\s*j\s*\]", head)
        assert not reads, (kernel, reads)


def test_no_function_is_left_that_nothing_calls():
    text = {f: source(f) for f in FILES}
    whole = "\n".join(text.values())
    names = {m[1] for f in ("paged.cuh", "paged_tc.cuh")
             for m in re.finditer(r"__device__ (?:__forceinline__ )?[\w:<> ]+?[\s*&](\w+)\((?!\()", text[f])}
    names |= {m[1] for f in ("paged.cuh", "paged_tc.cuh") for m in re.finditer(r"^(?:int|size_t|AttnPlan|constexpr uint32_t) (\w+)\(",
                                                                            text[f], re.M)}
    assert {"mbar_wait", "tmem_ld32", "peer_smem", "tokens", "launch_attention_many"} <= names
    unused = {n for n in names if len(re.findall(r"\b%s\b(?=\s*(?:<[\w:, ]+>)?\s*\()" % n, whole)) <
              1 + len(re.findall(r"(?:__forceinline__ [\w:<> ]+?[\s*&]|^(?:int|size_t|AttnPlan) )%s\(" % n, whole, re.M))}
    assert not unused
