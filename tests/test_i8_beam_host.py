"""Host side of the 8-bit unembedding and the beam search, without a GPU: refusals that need
no device, the layout of caches, and the restatement the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import i8_beam_ref as ref
from vindexllm_b200 import _lib, abi
from vindexllm_b200.build import build


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def test_null_handles_are_refused(lib):
    out = C.c_void_p()
    assert lib.vdxs_rms_norm_i8(None, None, 8, None, 0, 0, None, 0, 1, 8, 1e-6, None, 0, None, 8, None,
                                None) == abi.E_INVALID_ARG
    assert lib.vdxs_i8_prepare(None, None, 0, None, 8, 8, 8, None, C.byref(out)) == abi.E_INVALID_ARG
    assert lib.vdxs_unembed_i8(None, None, None, 16, None, 1, None, 0, 8, None) == abi.E_INVALID_ARG
    assert lib.vdxs_beam_create(None, 1, 1, 1, C.byref(out)) == abi.E_INVALID_ARG
    cfg, rows = abi.VdxsBeamConfig(), abi.VdxsBeamRows()
    assert lib.vdxs_beam_step(None, C.byref(cfg), None, 0, 1, C.byref(rows), C.byref(rows), None, 0, None, 0, None,
                              None, None) == abi.E_INVALID_ARG
    assert lib.vdxs_beam_reorder(None, None, None, 0, None) == abi.E_INVALID_ARG
    assert b"NULL" in lib.vdxs_last_error(None)
    assert lib.vdxs_i8_release(None) == abi.OK and lib.vdxs_beam_destroy(None) == abi.OK


def test_record_layouts():
    assert [getattr(abi.VdxsBeamConfig, n).offset for n, _ in abi.VdxsBeamConfig._fields_] == [0, 8, 12, 16, 20]
    assert [getattr(abi.VdxsBeamCache, n).offset for n, _ in abi.VdxsBeamCache._fields_] == list(range(0, 64, 8))


@pytest.mark.parametrize("shape,cut,want", [
    ((6, 5), None, (20, 20, 20, 1)),
    ((6, 4, 8, 16), None, (2048, 2048, 2048, 1)),
    ((6, 4, 8, 16), 3, (2048, 512, 192, 4)),
    ((6, 1, 8, 16), 3, (512, 192, 192, 1)),
    ((1, 4, 8, 16), 3, (2048, 512, 192, 4)),
])
def test_cache_pieces(shape, cut, want):
    import torch
    from vindexllm_b200.sampler import _cache_pieces
    t = torch.zeros(shape)
    assert _cache_pieces(t if cut is None else t[:, :, :cut], "cache") == want


def test_cache_pieces_at_no_single_distance():
    import torch
    from vindexllm_b200.sampler import _cache_pieces
    with pytest.raises(ValueError):
        _cache_pieces(torch.zeros(2, 3, 4, 5)[:, :, :2, :3], "cache")
    assert _cache_pieces(torch.zeros(2, 4, 6), "cache", 24) == (96, 24, 24, 4)


def test_restatement_against_the_definition():
    """Two beams over three tokens, worked by hand: probabilities 1/2, 1/4, 1/4."""
    x = np.log(np.array([[2, 1, 1], [1, 1, 2]], np.float32))
    s = dict(scores=np.array([0.0, -0.5], np.float32), lengths=np.array([0, 0], np.int32),
             finished=np.zeros(2, np.int32))
    tokens, parents, new, _, _ = ref.beam_step(x, 1, 2, s, (2,))
    assert tokens.tolist() == [[0, 2]] and parents.tolist() == [[0, 1]]
    assert np.allclose(new["scores"], [np.log(0.5), np.log(0.5) - 0.5]) and new["finished"].tolist() == [0, 1]
    q, scale = ref.norm_i8(np.array([[3.0, -4.0]]), np.ones(2), 0.0)
    assert q.tolist() == [[95, -127]] and np.allclose(scale * q[0, 1], -4 / np.sqrt(12.5))


def test_search_of_a_closed_context_is_refused():
    """A search's handle points to its context's: neither is used once the context is closed."""
    from types import SimpleNamespace

    from vindexllm_b200.sampler import BeamSearch, VdxsError
    search = BeamSearch.__new__(BeamSearch)
    search.ctx, search.lib, search._h = SimpleNamespace(_h=None, device=0), SimpleNamespace(), 1
    search.batch, search.beams, search.vocab = 1, 2, 10
    for call in (lambda: search.step(None, None), lambda: search.reorder(None, [])):
        with pytest.raises(VdxsError, match="context is closed"):
            call()
    search._h = None


def test_forms_of_the_product(tmp_path):
    """The rule that chooses the product's form, for the shapes that the GPU tests mean to reach each form
    with, at a B200's 148 SMs."""
    import os
    import shutil
    import subprocess

    from test_gpu_i8 import PAIR_SHAPES
    include = "/usr/local/cuda/include"
    if not shutil.which("g++") or not os.path.exists(os.path.join(include, "cuda_runtime.h")):
        pytest.skip("no g++ or CUDA headers")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / "form.cpp", tmp_path / "form"
    src.write_text('#include "vdxs_internal.h"\n#include <cstdio>\nint main() {\n int b, n, k;\n'
                   ' while (std::scanf("%d %d %d", &b, &n, &k) == 3) {\n'
                   '  const vdxs::I8ProductForm f = vdxs::i8_product_form(b, k, n, 148);\n'
                   '  std::printf("%d %d %d %d\\n", f.mode, f.split, f.n_tiles, f.n);\n }\n}\n')
    subprocess.run(["g++", "-std=c++17", "-I", include, "-I", os.path.join(root, "vindexllm_b200", "csrc"), str(src), "-o",
                    str(exe)], check=True)
    single = [(1, 262144, 1152), (64, 262144, 2560), (7, 20001, 2048), (256, 262144, 1152)]
    split = {(1, 1000, 8192): 8, (256, 1000, 8192): 8, (33, 8000, 4100): 2, (300, 700, 2000): 4}
    shapes = PAIR_SHAPES + single + list(split)
    run = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, s)) for s in shapes), capture_output=True, text=True,
                         check=True)
    got = {s: tuple(map(int, line.split())) for s, line in zip(shapes, run.stdout.splitlines())}
    assert all(got[s][0] == 1 for s in PAIR_SHAPES), got
    assert all(got[s][0] == 0 for s in single), got
    assert all(got[s][:2] == (2, parts) for s, parts in split.items()), got
    assert {got[s][3] for s in PAIR_SHAPES} >= {160, 256} and {got[s][2] for s in PAIR_SHAPES} >= {1, 2, 3}
    for (batch, _, _), (mode, _, n_tiles, n) in got.items():
        assert n_tiles * n >= batch and (n_tiles - 1) * n < batch and n <= 256 and n % (32 if mode == 1 else 16) == 0
