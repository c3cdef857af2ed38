"""Refusals of the rotary and differential-attention entries of the C-ABI, and the host-side helpers of their wrappers: no GPU needed.  Every
call here is one that the entry turns down before it launches anything; the pointers are never followed."""
import ctypes as C
import math

import pytest
import torch

P = 1 << 20  # stands for a 16-byte aligned device pointer; multiples of it for tensors that lie apart (each call's are smaller than that)


def _lib():
    from mofo_amd import _lib
    return _lib.load()


def _error():
    return _lib().mofo_last_error().decode()


def _rope(**kw):
    a = dict(x=P, bf=1, ldx=128, out=2 * P, ldo=128, M=4, heads=2, hd=64, freqs=3 * P, naxes=3, sections=(8, 12, 12, 0), pos=4 * P, tok=None, gh=14, gw=14, inter=0, inv=0)
    a.update(kw)
    s = (C.c_int * 4)(*a["sections"]) if a["sections"] is not None else None
    return _lib().mofo_rope_axes(a["x"], a["bf"], a["ldx"], a["out"], a["ldo"], a["M"], a["heads"], a["hd"], a["freqs"], a["naxes"], s, a["pos"], a["tok"], a["gh"],
                                 a["gw"], a["inter"], a["inv"], None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(out=None), dict(freqs=None), dict(sections=None), dict(M=0), dict(heads=0), dict(hd=0), dict(naxes=0), dict(naxes=5), dict(pos=None),
    dict(tok=P), dict(pos=None, tok=P, naxes=2, sections=(16, 16, 0, 0)), dict(pos=None, tok=P, gw=0), dict(sections=(-8, 20, 20, 0)), dict(sections=(8, 12, 13, 0)),
    dict(sections=(0, 0, 0, 0)), dict(sections=(12, 12, 16, 0)), dict(hd=60), dict(hd=2048, ldx=4096, ldo=4096), dict(ldx=120), dict(ldo=127), dict(ldx=132),
    dict(x=P + 2), dict(out=2 * P + 8), dict(out=P, ldo=136), dict(bf=0, ldx=130),
    dict(out=P + 16), dict(out=P + 128, ldx=256, ldo=256), dict(out=3 * P), dict(out=4 * P), dict(pos=None, tok=2 * P + 64)])
def test_rope_entry_refuses(bad):
    assert _rope(**bad) < 0 and "mofo_rope_axes" in _error()


def _fwd(**kw):
    a = dict(q=P, ldq=512, k=2 * P, ldk=256, v=3 * P, ldv=256, B=2, Nq=5, Nk=7, H=4, Hkv=2, scale=0.125, lam=5 * P, lam_heads=4, lam_init=0.4, gamma=None, pbf=1,
             eps=1e-5, out_scale=1.0, kv_len=None, causal=0, out=4 * P, ldo=512, o=None, o2=None, lse2=None, ws=None, n=0)
    a.update(kw)
    return _lib().mofo_diff_attention_fwd(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(lam=None), dict(out=None), dict(B=0), dict(Nq=0), dict(Nk=-1), dict(H=0), dict(Hkv=0), dict(Hkv=3), dict(scale=0.0),
    dict(scale=-0.5), dict(scale=math.nan), dict(scale=math.inf), dict(lam_heads=2), dict(causal=3), dict(causal=-1), dict(ldq=504), dict(ldk=128), dict(ldv=260),
    dict(ldk=1 << 25), dict(q=P + 8), dict(k=P + 2), dict(ldo=511), dict(out=P + 4), dict(o=6 * P), dict(o=6 * P, o2=7 * P), dict(lse2=8 * P),
    dict(o=6 * P + 8, o2=7 * P, lse2=8 * P), dict(out=P), dict(out=2 * P), dict(out=P + 1024, ldq=1024, ldo=1032), dict(o=6 * P, o2=6 * P + 64, lse2=8 * P),
    dict(o=6 * P, o2=7 * P, lse2=4 * P), dict(gamma=4 * P + 16), dict(kv_len=4 * P), dict(Nq=1, Nk=4096, ldk=256, ws=None), dict(Nq=1, Nk=4096, ws=9 * P, n=100),
    dict(scale=2.0 ** -25), dict(scale=2.0 ** 25), dict(gamma=20 * P, eps=0.0), dict(gamma=20 * P, eps=-1e-5), dict(gamma=20 * P, eps=math.nan),
    dict(H=8192, ldq=1 << 20, ldo=1 << 20, lam_heads=1), dict(B=1 << 20, Nk=1 << 20), dict(Nq=1 << 30)])
def test_diff_attention_entry_refuses(bad):
    assert _fwd(**bad) < 0 and "mofo_diff_attention_fwd" in _error()


def _bwd(**kw):
    a = dict(q=P, ldq=512, k=2 * P, ldk=256, v=3 * P, ldv=256, B=2, Nq=5, Nk=7, H=4, Hkv=2, scale=0.125, lam=4 * P, lam_heads=4, lam_init=0.4, gamma=None, pbf=1,
             eps=1e-5, out_scale=1.0, kv_len=None, causal=0, o=5 * P, o2=6 * P, lse2=7 * P, dout=8 * P, lddo=512, dq=9 * P, lddq=512, dk=10 * P, lddk=256,
             dv=11 * P, lddv=256, dlam=12 * P, dgamma=None, gbf=1, ws=13 * P, n=1 << 30)
    a.update(kw)
    return _lib().mofo_diff_attention_bwd(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(o=None), dict(o2=None), dict(lse2=None), dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(dlam=None), dict(ws=None), dict(n=10),
    dict(gamma=20 * P), dict(dgamma=20 * P), dict(dq=P), dict(dk=3 * P), dict(dv=10 * P + 128), dict(dlam=4 * P), dict(ws=8 * P), dict(dq=5 * P), dict(lddo=504), dict(lddq=256), dict(lddk=130), dict(lddv=128), dict(dout=8 * P + 8), dict(ws=13 * P + 4), dict(H=5), dict(q=None),
    dict(lddo=1 << 25), dict(scale=2.0 ** -25), dict(gamma=30 * P, dgamma=31 * P, eps=0.0)])
def test_diff_attention_gradient_entry_refuses(bad):
    assert _bwd(**bad) < 0 and "mofo_diff_attention_bwd" in _error()


def test_scratch_sizes():
    lib = _lib()
    for f, tail in ((lib.mofo_diff_attention_fwd_ws, ()), (lib.mofo_diff_attention_bwd_ws, (1,))):
        assert f(0, 5, 5, 4, 2, *tail) < 0 and f(1, 5, 5, 4, 3, *tail) < 0
        assert f(1, 1, 1, 1, 1, *tail) >= 0
    # the gradient's: four statistics a row and head, the rows behind the norm in bf16, and what a block of rows leaves for the parameters
    assert lib.mofo_diff_attention_bwd_ws(32, 1568, 1568, 3, 3, 1) >= 32 * 1568 * 3 * (4 + 64)
    assert lib.mofo_diff_attention_bwd_ws(32, 1568, 1568, 3, 3, 1) - lib.mofo_diff_attention_bwd_ws(32, 1568, 1568, 3, 3, 0) == 32 * 1568 * 3 * 64


def test_wrappers_refuse_the_cpu():
    from mofo_amd import ops
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), ops.rope_freqs((8, 12, 12), device="cpu"), x.clone(), pos=torch.zeros(4, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        ops.diff_attention_fwd(x, x, x, 1, 1, 1, 0.125, torch.zeros(4, 1, 64), 0.4, x.clone())


def test_rope_frequencies():
    from mofo_amd import ops
    f = ops.rope_freqs((2, 3, 1), 100.0, "cpu")
    want = [1.0, 100.0 ** -0.5, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3), 1.0]
    assert f.dtype == torch.float64 and torch.allclose(f * 2 * math.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-15, atol=0)
    assert ops.rope_freqs((0, 8, 0), device="cpu").numel() == 8


BIG = 1 << 36   # as P, for tensors of many GiB


@pytest.mark.parametrize("bad", [
    dict(M=1 << 27, heads=1, hd=16, ldx=16, ldo=16, naxes=1, sections=(8, 0, 0, 0)), dict(M=(1 << 27) + 1, heads=2, hd=64, bf=0),
    dict(M=1 << 26, heads=16, hd=64, ldx=1024, ldo=1024), dict(M=1 << 30, heads=1, hd=64, ldx=64, ldo=64)])
def test_rope_entry_refuses_more_blocks_than_a_launch_takes(bad):
    """2^24 blocks of 256 threads are 2^32 threads, one more than a launch counts"""
    a = dict(x=BIG, out=8 * BIG, freqs=P, pos=16 * BIG)
    assert _rope(**{**a, **bad}) < 0 and "blocks" in _error()


MANY = [dict(B=1 << 20, Nq=1, Nk=1, H=16, Hkv=16), dict(B=1 << 24, Nq=1, Nk=1, H=1, Hkv=1), dict(B=1 << 22, Nq=1, Nk=1, H=8, Hkv=4), dict(B=1 << 20, Nq=17, Nk=17, H=16, Hkv=16)]


@pytest.mark.parametrize("bad", MANY)
def test_diff_attention_entry_refuses_more_blocks_than_a_launch_takes(bad):
    w = bad["H"] * 128
    a = dict(q=BIG, ldq=w, k=4 * BIG, ldk=w, v=8 * BIG, ldv=w, out=12 * BIG, ldo=w, lam_heads=1)
    assert _fwd(**{**a, **bad}) < 0 and "mofo_diff_attention_fwd" in _error() and "blocks" in _error()


@pytest.mark.parametrize("bad", MANY + [dict(B=1 << 19, Nq=1, Nk=1, H=16, Hkv=16)])
def test_diff_attention_gradient_entry_refuses_more_blocks_than_a_launch_takes(bad):
    """dK / dV, dQ and the parameters' blocks are one launch: half as many (clip, key head) pairs fill it"""
    w = bad["H"] * 128
    a = dict(q=BIG, ldq=w, k=4 * BIG, ldk=w, v=8 * BIG, ldv=w, lam_heads=1, o=12 * BIG, o2=16 * BIG, lse2=20 * BIG, dout=24 * BIG, lddo=w, dq=28 * BIG, lddq=w,
             dk=32 * BIG, lddk=w, dv=36 * BIG, lddv=w, ws=40 * BIG, n=1 << 40)
    assert _bwd(**{**a, **bad}) < 0 and "mofo_diff_attention_bwd" in _error() and "blocks" in _error()


def test_wrappers_refuse_pitches_that_do_not_fit_the_entries():
    """the C entries take row pitches as 32-bit ints: a pitch of 2^32 + 512 elements is not one of 512"""
    from mofo_amd import ops
    for pitch, ok in ((512, True), ((1 << 31) - 8, True), (1 << 31, False), ((1 << 32) + 512, False)):
        t = torch.empty_strided((2, 128), (pitch, 1), dtype=torch.bfloat16, device="meta")
        if ok:
            assert ops._pitch(-1, torch.bfloat16, "q", t) == pitch
        else:
            with pytest.raises(ValueError, match="pitch"):
                ops._pitch(-1, torch.bfloat16, "q", t)
