"""What the norms', gated activations' and adapters' host and device sources have to keep to, on the CPU."""

from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from moss_offload import _native, adapters, gated, kept8, norms

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"mo_norm_call": (_native.MoNormCall, norms._CALL), "mo_gated_call": (_native.MoGatedCall, gated._CALL),
           "mo_adapters_call": (_native.MoAdaptersCall, adapters._CALL)}


def test_the_calls_lie_as_the_header_says(tmp_path) -> None:
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "moss_offload.h"}"', "int main(void) {"]
    for name, (cls, _) in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));' for field, _ in cls._fields_]
    source, exe = tmp_path / "calls.c", tmp_path / "calls"
    source.write_text("\n".join([*lines, "return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(source)], check=True)
    said = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, (cls, packed) in STRUCTS.items():
        assert int(said[name]) == ctypes.sizeof(cls) == packed.size, name
        for field, _ in cls._fields_:
            assert int(said[f"{name}.{field}"]) == getattr(cls, field).offset, field


def test_wide_stores_have_no_scalar_offset() -> None:
    """With a register there, the compiler lets the next instruction overwrite what the store has yet to read."""

    seen = 0
    for path in sorted((ROOT / "moss-image_amd" / "csrc").glob("*")):
        for call in re.findall(r"raw_buffer_store_b(?:96|128)\((.*?)\);", path.read_text(), flags=re.S):
            seen += 1
            assert re.search(r",\s*0,\s*[^,]+$", call), (path.name, call)
    assert seen


def test_a_checkpoint_that_a_graph_captures_is_refused(monkeypatch) -> None:
    class Tokens(torch.Tensor):
        is_cuda = True

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        kept8.checkpoint_kept8(lambda t: t, torch.zeros(2, 32, requires_grad=True).as_subclass(Tokens))
