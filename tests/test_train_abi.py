"""CPU checks of the trainable block pieces' interface: the records that the
Python and the Rust binding mirror have the layout of the C header, the entry
points refuse NULL contexts, and the wrappers refuse tensors that are not on a
GPU before anything is launched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch
import vestra_kernels as vk

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FFI = os.path.join(ROOT, "vestra-kernels_b200", "bindings", "rust", "src", "b200", "ffi.rs")
RECORDS = {
    "vk_heads": ("_Heads", "VkHeads"),
    "vk_attention_shape": ("_AttentionShape", "VkAttentionShape"),
    "vk_rope_axes_shape": ("_RopeAxesShape", "VkRopeAxesShape"),
    "vk_residual_norm_shape": ("_ResidualNormShape", "VkResidualNormShape"),
    "vk_residual_norm_grads": ("_ResidualNormGrads", "VkResidualNormGrads"),
}


@pytest.fixture(scope="module")
def layouts(tmp_path_factory):
    """{record: {field: (offset, size)}} and {record: size}, from a C program that includes the header."""
    d = tmp_path_factory.mktemp("abi")
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "vestra_b200.h"', "int main(void) {"]
    for record, (py, _) in RECORDS.items():
        lines.append(f'  printf("{record} . %zu 0\\n", sizeof({record}));')
        for field, _ in getattr(vk, py)._fields_:
            lines.append(f'  printf("{record} {field} %zu %zu\\n", offsetof({record}, {field}), sizeof((({record}*)0)->{field}));')
    (d / "layout.c").write_text("\n".join(lines + ["  return 0;", "}", ""]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(d / "layout.c"), "-o",
                    str(d / "layout")], check=True)
    fields, sizes = {r: {} for r in RECORDS}, {}
    for line in subprocess.run([str(d / "layout")], capture_output=True, text=True, check=True).stdout.splitlines():
        record, field, a, b = line.split()
        if field == ".":
            sizes[record] = int(a)
        else:
            fields[record][field] = (int(a), int(b))
    return fields, sizes


@pytest.mark.parametrize("record", RECORDS)
def test_python_records_are_the_headers(layouts, record):
    fields, sizes = layouts
    struct = getattr(vk, RECORDS[record][0])
    assert ctypes.sizeof(struct) == sizes[record]
    for name, _ in struct._fields_:
        d = getattr(struct, name)
        assert (d.offset, d.size) == fields[record][name], name


RUST_SIZES = {"c_int": 4, "f32": 4, "usize": 8, "i64": 8}


@pytest.mark.parametrize("record", RECORDS)
def test_rust_records_are_the_headers(layouts, record):
    """Fields in the header's order with the header's sizes; repr(C) then gives the header's offsets."""
    src = open(FFI).read()
    axes = int(re.search(r"pub const VK_ROPE_MAX_AXES: usize = (\d+)", src).group(1))
    body = re.search(r"#\[repr\(C\)\]\s*pub struct %s \{(.*?)\}" % RECORDS[record][1], src, re.S).group(1)
    rust = []
    for name, kind in re.findall(r"pub (\w+): ([^,;\[\]]+(?:\[[^\]]*\])?|\[[^\]]*\])", body):
        kind = kind.strip()
        if kind.startswith("*"):
            size = 8
        elif kind.startswith("["):
            size = axes * RUST_SIZES[kind[1:].split(";")[0]]
        else:
            size = RUST_SIZES[kind]
        rust.append((name, size))
    fields, _ = layouts
    assert rust == [(n, s) for n, (o, s) in sorted(fields[record].items(), key=lambda f: f[1][0])]


def test_axes_limit_is_the_headers():
    text = open(os.path.join(ROOT, "include", "vestra_b200.h")).read()
    assert int(re.search(r"#define VK_ROPE_MAX_AXES (\d+)", text).group(1)) == vk.ROPE_MAX_AXES


@pytest.mark.parametrize("name", ["vk_attention_forward", "vk_attention_backward", "vk_rope_axes", "vk_residual_norm_forward",
                                  "vk_residual_norm_backward", "vk_residual_norm_workspace"])
def test_null_contexts_are_refused(name):
    fn = getattr(vk.lib(), name)
    args = [None if t in (ctypes.c_void_p,) or not issubclass(t, ctypes._SimpleCData) else 0 for t in fn.argtypes]
    assert fn(*args) == vk.VK_ERR_INVALID_ARGUMENT
    assert "NULL context" in vk.last_error()


def test_wrappers_refuse_tensors_off_the_gpu():
    x = torch.zeros(1, 2, 3, 64)
    lse, rows = torch.zeros(1, 2, 3), torch.zeros(1, 3, 8)
    vec, stats = torch.zeros(8), torch.zeros(1, 3, 2)
    pos = torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: vk.attention_forward(x, x, x, x, lse),
                 lambda: vk.attention_backward(x, x, x, x, lse, x, x, x, x),
                 lambda: vk.rope_axes(x, x, pos, (32, 32), 100.0, x, x),
                 lambda: vk.residual_norm_forward(rows, rows, vec, vec, 1e-6, rows, rows, stats),
                 lambda: vk.residual_norm_workspace(rows, rows),
                 lambda: vk.residual_norm_backward(rows, rows, rows, rows, stats, vec, rows, rows, vec, vec)):
        with pytest.raises(TypeError, match="CUDA"):
            call()
