"""CPU: a MultiAxisRotary, and a module that holds one, can be copied, pickled and saved."""

from __future__ import annotations

import copy
import io
import pickle
import subprocess
import sys

import pytest
import torch

import tilelang_fa2_4d_mask as api
from conftest import ROOT
from fa2_with_4d_mask_b200 import _lib


def rope():
    return api.MultiAxisRotary(96, (10, 0, 22), base=5e5, rotary_dim=64, pairing="adjacent")


def same(a, b):
    assert type(a) is type(b) and a is not b
    for name in ("head_dim", "sections", "base", "rotary_dim", "pairing"):
        assert getattr(a, name) == getattr(b, name)
    assert _lib.host().table_turns(a._table) == _lib.host().table_turns(b._table)


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy] + [lambda x, p=p: pickle.loads(pickle.dumps(x, p)) for p in range(2, 6)])
def test_copies(how):
    a = rope()
    a.note = [1]
    b = how(a)
    same(a, b)
    assert b.note == [1]
    # And it runs as far as the device.
    x = torch.zeros(1, 1, 2, 96, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        b(x, x, torch.zeros(3, 1, 2, dtype=torch.int64))


def test_a_module_that_holds_one():
    m = torch.nn.Linear(2, 2)
    m.rotary = rope()
    same(m.rotary, copy.deepcopy(m).rotary)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    same(m.rotary, torch.load(f, weights_only=False).rotary)


def test_a_process_that_has_not_imported_the_package(tmp_path):
    path = tmp_path / "rope.pkl"
    path.write_bytes(pickle.dumps(rope()))
    code = f"import pickle; r = pickle.load(open({str(path)!r}, 'rb')); print(r.sections, r.base, r.pairing)"
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert out.stdout.strip() == "(10, 0, 22) 500000.0 adjacent"
