"""The rule of overlapping launches, checked on the sources: a kernel that may become resident while the one
before it still runs waits for it (``pdl_wait``) on every thread, unconditionally, before it reads anything that an
earlier kernel may have written, and before the first of its bounded waits, whose budget is meant for its own work."""

import glob
import os
import re

import pytest

import lucid_b200

CSRC = os.path.join(os.path.dirname(lucid_b200.__file__), "csrc")
ACCESS = re.compile(r"__ldg|__ldcg|\bld\.global|\bindex_at\(|\.load\(|\bload_\w+\(|\btma_load|\bmbar_wait|\bflag_wait|\batomic")
NAMED = re.compile(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(")


def _kernels():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in NAMED.finditer(text):
            begin = text.index("{", m.end())
            end, depth = begin + 1, 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            body = text[begin + 1:end - 1]
            if "pdl_wait();" in body:
                yield f"{os.path.basename(path)}:{m.group(1)}", body


KERNELS = dict(_kernels())
OVERLAPPING = ["gemm_s8.cu:gemm_s8_kernel", "kvcache.cu:kv_mark_kernel", "kvcache.cu:kv_write_kernel",
               "kvcache.cu:kv_read_kernel", "microscale.cu:mx_quantize_kernel", "gemm_mx.cu:mx_pair_kernel",
               "gemm_mx.cu:mx_tile_kernel"]


def test_the_scan_finds_the_kernels():
    assert set(OVERLAPPING) <= set(KERNELS)


@pytest.mark.parametrize("name", OVERLAPPING)
def test_nothing_is_read_before_the_wait(name):
    before = KERNELS[name].split("pdl_wait();")[0]
    assert ACCESS.findall(before) == []


@pytest.mark.parametrize("name", OVERLAPPING)
def test_every_thread_waits(name):
    before = KERNELS[name].split("pdl_wait();")[0]
    assert before.count("{") == before.count("}")          # not inside a branch
    assert before.rstrip()[-1:] in ("", ";", "}")           # nor behind a condition
