"""CPU: what adamw_step refuses, the argument structures against the header, the 8-bit format's arithmetic."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import adamw_cases as ac

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
RECORDS = {"AdamWTensor": "fdgs_adamw_tensor", "AdamWArgs": "fdgs_adamw_args", "Moment8Tensor": "fdgs_moment8_tensor",
           "Moment8Args": "fdgs_moment8_args", "EmbeddingFwdArgs": "fdgs_embedding_fwd_args",
           "EmbeddingBwdArgs": "fdgs_embedding_bwd_args"}


def test_records_match_the_header(tmp_path):
    """sizeof and the offset of every field against a C program; the packed formats against the structures."""
    from fdgs import _records
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    declared = {n for n, t in vars(_records).items() if isinstance(t, type) and issubclass(t, C.Structure)}
    assert declared == set(RECORDS)
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fdgs.h"', 'int main(void) {']
    for name, cname in RECORDS.items():
        lines.append(f'printf("{name} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in getattr(_records, name)._fields_]
    lines.append('printf("block x %d\\ntokens x %d\\n", FDGS_MOMENT8_BLOCK, FDGS_EMBEDDING_MAX_TOKENS); return 0; }')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")[:-1]
    for name, field, value in (line.split() for line in out):
        if name in ("block", "tokens"):
            assert int(value) == (_records.MOMENT8_BLOCK if name == "block" else _records.EMBEDDING_MAX_TOKENS)
            continue
        t = getattr(_records, name)
        assert int(value) == (C.sizeof(t) if field == "sizeof" else getattr(t, field).offset), (name, field)


def test_library_refuses_what_it_cannot_step():
    from fdgs import _lib, _records
    lib = _lib.lib

    def rc(count=1, kind=0, bits=32, betas=(0.9, 0.999), eps=1e-8, **over):
        f = dict(param=64, grad=64, exp_avg=64, exp_avg_sq=64, numel=4, step=1, lr=1e-3)
        f.update(over)
        rec = bytes(_records.AdamWTensor(**f))
        return lib.fdgs_adamw_step(C.byref(_records.AdamWArgs(count, kind, bits, 0, *betas, eps, rec)), None)
    assert lib.fdgs_adamw_step(None, None) == -1
    assert rc(count=-1) == -1 and rc(kind=2) == -1 and rc(bits=16) == -1
    assert rc(betas=(1.0, 0.9)) == -1 and rc(betas=(0.9, float("nan"))) == -1 and rc(eps=-1.0) == -1
    assert rc(step=0) == -1 and rc(numel=-1) == -1 and rc(grad_row_len=4, grad_row_stride=3) == -1 and rc(grad_row_len=-1) == -1
    for name in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert rc(**{name: 0}) == -1
    assert rc(kind=1) == -1                      # bfloat16 without a residual
    assert rc(bits=8) == -1 and rc(bits=8, exp_avg_exponents=64) == -1 and rc(bits=8, exp_avg_sq_exponents=64) == -1
    assert rc(numel=1 << 50) == -4
    assert rc(count=0) == 0 and rc(numel=0, param=0) == 0         # nothing to do
    assert lib.fdgs_adamw_step(C.byref(_records.AdamWArgs(1, 0, 32, 0, 0.9, 0.9, 0.0, None)), None) == -1

    def m8(name, count=1, kind=0, nearest=1, **over):
        f = dict(codes=64, exponents=64, value=64, numel=4, is_signed=1)
        f.update(over)
        rec = bytes(_records.Moment8Tensor(**f))
        return getattr(lib, name)(C.byref(_records.Moment8Args(count, kind, nearest, 0, rec)), None)
    for name in ("fdgs_moment8_pack", "fdgs_moment8_unpack"):
        assert m8(name, count=-1) == -1 and m8(name, kind=2) == -1 and m8(name, numel=-1) == -1
        for field in ("codes", "exponents", "value"):
            assert m8(name, **{field: 0}) == -1
        assert m8(name, numel=0) == 0 and m8(name, numel=1 << 50) == -4
    assert m8("fdgs_moment8_pack", kind=1) == -1                  # packs float32 values only


def test_step_refuses_its_arguments_before_any_launch():
    from fdgs import adamw
    p, g, m, v = (torch.zeros(8) for _ in range(4))
    with pytest.raises(RuntimeError, match="GPU only"):
        adamw.adamw_step([p], [g], [m], [v], steps=1, lr=1e-3)
    with pytest.raises(ValueError, match="same length"):
        adamw.adamw_step([p], [g], [m], [], steps=1, lr=1e-3)
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        adamw.adamw_step([p.half()], [g], [m], [v], steps=1, lr=1e-3)
    with pytest.raises(ValueError, match="each of the 1"):
        adamw.adamw_step([p], [g], [m], [v], steps=[1, 2], lr=1e-3)
    assert adamw.adamw_step([], [], [], [], steps=1, lr=1e-3) is None
    with pytest.raises(RuntimeError, match="GPU only"):
        adamw.pack8([p], True)
    with pytest.raises(ValueError, match="one for each"):
        adamw.pack8([p], [True, False])
    assert adamw.pack8([], True) == [] and adamw.unpack8([]) == []


def test_hash_is_even_and_keys_are_apart():
    """Both halves of the hash over 2^18 consecutive indices: 64 cells' counts within five deviations, means of the bits
    likewise, and neither half correlated between neighbouring elements or steps."""
    from fdgs import adamw
    n = 1 << 18
    keys = [adamw.round_key(s, i, t) for s in (0, 1) for i in (0, 1, 39) for t in (1, 2, 1000)]
    assert len(set(keys)) == len(keys) and all(0 <= k < 1 << 32 for k in keys)
    rows = [ac.hash32(np.arange(n), k) for k in keys]
    for h in rows:
        for half in (h >> 16, h & 0xFFFF):
            count = np.bincount(half >> 10, minlength=64)
            assert np.abs(count - n / 64).max() <= 5 * np.sqrt(n / 64)
            x = half / 32768.0 - 1.0
            assert abs(np.mean(x[1:] * x[:-1])) * 3 <= 5 / np.sqrt(n)
    for a, b in zip(rows, rows[1:]):
        x, y = (a & 0xFFFF) / 32768.0 - 1.0, (b & 0xFFFF) / 32768.0 - 1.0
        assert abs(np.mean(x * y)) * 3 <= 5 / np.sqrt(n)


def test_split_of_a_weight_is_exact():
    rng = np.random.default_rng(1)
    w = (rng.standard_normal(10000) * 10.0 ** rng.uniform(-30, 30, 10000)).astype(np.float32)
    w[:3] = 0.0, -0.0, np.float32(1.00390625)            # zero both ways, halfway between two bfloat16 numbers
    hi, lo = ac.split_bf16(w)
    back = ((hi.astype(np.int64) << 16) + lo.astype(np.int64)).astype(np.uint32).view(np.float32)
    assert np.array_equal(back.view(np.uint32), w.view(np.uint32))


def test_optimizer_refuses_what_it_does_not_do():
    from fdgs.adamw import FusedAdamW
    p = torch.zeros(4, requires_grad=True)
    for bad, match in ((dict(state_bits=16), "8 or 32"), (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "betas")):
        with pytest.raises(ValueError, match=match):
            FusedAdamW([p], **bad)
    for key in ("amsgrad", "maximize"):
        with pytest.raises(ValueError, match="amsgrad"):
            FusedAdamW([{"params": [p], key: True}])
    with pytest.raises(ValueError, match="twice"):
        FusedAdamW([{"params": [p]}, {"params": [p]}])
    opt = FusedAdamW([p])
    opt.step()                                   # nothing has a gradient
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU only"):
        opt.step()
    assert opt.state == {} and opt.state_dict()["state"] == {}
    with pytest.raises(ValueError, match="different parameter groups"):
        opt.load_state_dict({"state": {}, "param_groups": []})
    opt.zero_grad(set_to_none=False)
    assert (p.grad == 0).all()
    half = torch.zeros(4, dtype=torch.float16)
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        FusedAdamW([half])._new_state(half)


def test_steps_and_conversions_that_no_grid_holds_are_refused():
    """A launch has fewer than 2^32 threads: 2^23 workgroups of 512 for 2048 elements each, 2^24 of 256 for 4096."""
    from fdgs import _lib, _records
    lib = _lib.lib
    for each, most in ((2048, 1 << 23), (4096, 1 << 24)):
        for sizes in ([each * most], [each * most - each + 1], [each * most // 2, each * most // 2 - 5], [each * (most - 1), 1]):
            n = len(sizes)
            if each == 2048:
                recs = (_records.AdamWTensor * n)(*[_records.AdamWTensor(param=64, grad=64, exp_avg=64, exp_avg_sq=64, numel=k, step=1) for k in sizes])
                assert lib.fdgs_adamw_step(C.byref(_records.AdamWArgs(n, 0, 32, 0, 0.9, 0.9, 0.0, C.cast(recs, C.c_char_p))), None) == -4
                continue
            for name in ("fdgs_moment8_pack", "fdgs_moment8_unpack"):
                recs = (_records.Moment8Tensor * n)(*[_records.Moment8Tensor(codes=64, exponents=64, value=64, numel=k) for k in sizes])
                assert getattr(lib, name)(C.byref(_records.Moment8Args(n, 0, 1, 0, C.cast(recs, C.c_char_p))), None) == -4


def test_a_weight_decay_of_another_kind_is_not_taken_over():
    """Adam adds it to the gradient, AdamW takes it off the weight: the number means another step."""
    from fdgs.adamw import FusedAdamW
    p = torch.zeros(4, requires_grad=True)
    opt = FusedAdamW([p], weight_decay=0.3)
    with pytest.raises(ValueError, match="part of the gradient"):
        opt.load_state_dict(torch.optim.Adam([p], weight_decay=0.1).state_dict())
    assert opt.param_groups[0]["weight_decay"] == 0.3
    opt.load_state_dict(torch.optim.AdamW([p], weight_decay=0.2).state_dict())
    assert opt.param_groups[0]["weight_decay"] == 0.2
    opt.load_state_dict(torch.optim.Adam([p]).state_dict())
    assert opt.param_groups[0]["weight_decay"] == 0 and opt.param_groups[0]["decoupled_weight_decay"]
