"""Refusals of the serving operators: argument checks that run before any device work. They run
where there is no GPU only: the pointers are stand-ins, and a call that were accepted by mistake
must not reach a device."""

import pytest
import torch

from orchard_b200 import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers stand for nothing: no GPU may see them")

P = 4096  # stands for a 16-byte aligned device pointer: never read, the checks come first


def attention(**kw):
    a = dict(q=P, kp=P, vp=P, units=P, nu=1, mp=8, pcap=8, np_=1, kc=P, vc=P, lens=P, slots=None, mo=8, cap=8, ns=1, mass=None,
             out=P, M=1, nh=4, nkv=2, hd=64, ws=None, wb=0, st=None)
    a.update(kw)
    return _lib.lib().orch_attention_prefix(*a.values())


def evict(**kw):
    a = dict(k=P, v=P, mass=P, pos=P, lens=P, slots=None, mo=P, po=P, lo=2 * P, M=1, nkv=1, hd=64, cap=8, ns=1, budget=4, recent=1,
             st=None)
    a.update(kw)
    return _lib.lib().orch_cache_evict(*a.values())


def logits(**kw):
    a = dict(x=P, out=P, dt=0, M=1, V=10, ld=10, base=0, hist=None, hl=0, hn=None, gs=None, pen=None, bi=None, bv=None, bo=None,
             nb=0, masks=None, mw=0, nm=0, mr=None, st=None)
    a.update(kw)
    return _lib.lib().orch_logits_process(*a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), b"null"), (dict(kc=None), b"null"), (dict(lens=None), b"null"), (dict(out=None), b"null"),
    (dict(kp=None), b"null prefix"), (dict(units=None), b"null prefix"), (dict(nkv=3), b"multiple"), (dict(nkv=0), b"multiple"),
    (dict(hd=48), b"head_dim"), (dict(hd=256), b"head_dim"), (dict(mo=9), b"max_own"), (dict(ns=0), b"cache shape"),
    (dict(cap=0, mo=0), b"cache shape"), (dict(cap=2 ** 30), b"cache shape"), (dict(mp=9), b"max_prefix"),
    (dict(np_=0), b"prefix shape"), (dict(nu=2), b"units"), (dict(q=P + 2), b"aligned"), (dict(units=P + 4), b"aligned"), (dict(ws=P + 8, wb=1 << 30), b"aligned"),
    (dict(ws=None, mo=4000, cap=4000), b"workspace"), (dict(ws=P, wb=16, mo=4000, cap=4000), b"workspace")])
def test_attention_refusals(kw, word):
    assert attention(**kw) == 1 and word in _lib.lib().orch_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(k=None), b"null"), (dict(mo=None), b"null"), (dict(lo=None), b"null"), (dict(nkv=0), b"empty"), (dict(cap=0), b"empty"),
    (dict(ns=0), b"empty"), (dict(hd=12), b"head_dim"), (dict(hd=0), b"head_dim"), (dict(k=P + 8), b"aligned"),
    (dict(mo=2 * P), b"both"), (dict(po=2 * P), b"both"), (dict(lo=P), b"lens_out")])
def test_evict_refusals(kw, word):
    assert evict(**kw) == 1 and word in _lib.lib().orch_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(x=None), b"null"), (dict(out=None), b"null"), (dict(V=0), b"empty"), (dict(dt=2), b"dtype"), (dict(ld=9), b"stride"), (dict(ld=1 << 31), b"stride"),
    (dict(base=2 ** 31 - 5), b"range"), (dict(hist=P), b"penalties"), (dict(pen=P), b"penalties"), (dict(hist=P, pen=P), b"penalties"),
    (dict(bi=P), b"bias"), (dict(bi=P, bv=P), b"bias"), (dict(masks=P, mw=1, nm=1), b"masks"), (dict(masks=P, mr=P), b"masks"),
    (dict(M=65536), b"rows")])
def test_logits_refusals(kw, word):
    assert logits(**kw) == 1 and word in _lib.lib().orch_last_error()


def test_unsupported_shapes_and_empty_calls():
    L = _lib.lib()
    assert evict(cap=1000001) == 3 and b"1,000,000" in L.orch_last_error()
    assert attention(M=2 ** 31, nh=2, nkv=2) == 3
    assert attention(M=0, q=None) == 0 and evict(M=0, k=None) == 0 and logits(M=0, x=None) == 0


def test_workspace_size():
    f = _lib.lib().orch_attention_prefix_workspace_bytes
    assert f(0, 4, 4, 64, 1, 100, 100, 0) == 0 and f(1, 4, 3, 64, 1, 100, 100, 0) == 0
    assert f(1, 2, 2, 32, 1, 24, 8, 0) == 0  # one launch, nothing to join
    assert f(64, 32, 32, 128, 1, 4096, 640, 0) > 64 * 32 * 128 * 4
    assert f(64, 32, 32, 128, 1, 4096, 640, 1) >= f(64, 32, 32, 128, 1, 4096, 640, 0) + 64 * 32 * 640 * 4
