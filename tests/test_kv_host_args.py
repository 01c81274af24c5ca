"""The KV cache operators' Python layer refuses what is no memory of the context's GPU, before the library is called: its
address would go to the kernels. Needs no GPU: tensors that claim to be on one stand in for those that are right."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


class Claims:
    """a host tensor that says that it is on GPU `index`"""

    def __init__(self, t, index=0):
        self.t, self.index = t, index

    def get_device(self):
        return self.index

    def __getattr__(self, name):
        return getattr(self.t, name)


class Ctx:
    """a context without a library handle: a call that gets as far as the library is refused there for its null argument"""
    h, device = None, 0


def tensors(n_slot=2, n_kv=2, n_rows=16, d=128):
    q = [torch.zeros(n_slot, n_kv, n_rows, d, dtype=torch.int8) for _ in "kv"]
    return q + [torch.zeros(n_slot, n_kv, n_rows, d // 32, dtype=torch.float16) for _ in "kv"]


def calls(ocr, ctx, cache):
    """every operator with its tensor arguments, by name"""
    def rows(heads):
        return torch.zeros(2, 3, heads, 128)

    ints = dict(pos=torch.zeros(2, dtype=torch.int32), n=torch.zeros(2, dtype=torch.int32))
    tree = torch.zeros(2, 3, dtype=torch.int32)
    return [
        (lambda k, v, pos, n: ocr.op_kv_write(ctx, cache, k, v, pos, n), dict(k=rows(2), v=rows(2), **ints)),
        (lambda k, v, pos, n: ocr.op_kv_read(ctx, cache, k, v, pos, n), dict(k=rows(2), v=rows(2), **ints)),
        (lambda q, out, pos, n: ocr.op_attention_window(ctx, cache, q, out, pos, 0.1, n), dict(q=rows(4), out=rows(4), **ints)),
        (lambda q, out, pos, parent, n: ocr.op_attention_tree(ctx, cache, q, out, pos, parent, 0.1, n),
         dict(q=rows(4), out=rows(4), parent=tree, **ints)),
        (lambda pos, path, n: ocr.op_kv_keep(ctx, [cache, cache], pos, path, n), dict(path=tree, **ints)),
    ]


@pytest.mark.parametrize("which", range(4))
def test_a_cache_in_host_memory_is_refused(ocr, which):
    t = [Claims(x) for x in tensors()]
    ocr.KvCache("q8_0", *t)
    t[which] = t[which].t
    with pytest.raises(ocr.OcrError, match="device tensors"):
        ocr.KvCache("q8_0", *t)
    t[which] = Claims(t[which], 1)
    with pytest.raises(ocr.OcrError, match="on GPU"):
        ocr.KvCache("q8_0", *t)


@pytest.mark.parametrize("op", range(5))
def test_arguments_in_host_memory_or_on_another_gpu_are_refused(ocr, op):
    cache = ocr.KvCache("q8_0", *(Claims(x) for x in tensors()))
    call, args = calls(ocr, Ctx(), cache)[op]
    good = {k: Claims(v) for k, v in args.items()}
    with pytest.raises(ocr.OcrError, match="null argument"):  # (nothing else is wrong with them)
        call(**good)
    for name in args:
        with pytest.raises(ocr.OcrError, match="device tensors"):
            call(**{**good, name: args[name]})
        with pytest.raises(ocr.OcrError, match="device tensors"):
            call(**{**good, name: args[name].numpy()})
        with pytest.raises(ocr.OcrError, match="on GPU 1"):
            call(**{**good, name: Claims(args[name], 1)})


@pytest.mark.parametrize("op", range(5))
def test_a_cache_on_another_gpu_than_the_context_is_refused(ocr, op):
    cache = ocr.KvCache("q8_0", *(Claims(x, 1) for x in tensors()))
    call, args = calls(ocr, Ctx(), cache)[op]
    with pytest.raises(ocr.OcrError, match="the context on GPU 0"):
        call(**{k: Claims(v, 1) for k, v in args.items()})


@pytest.mark.parametrize("op", range(5))
def test_the_cache_of_a_closed_session_is_refused(ocr, op):
    """its rows' memory went with the session"""
    session = SimpleNamespace(h=1, model=SimpleNamespace(ctx=Ctx()))
    cache = ocr.KvCache._of(ocr.KvCache("q8_0", *(Claims(x) for x in tensors())).c, session)
    call, args = calls(ocr, Ctx(), cache)[op]
    args = {k: Claims(v) for k, v in args.items()}
    with pytest.raises(ocr.OcrError, match="null argument"):
        call(**args)
    session.h = None
    with pytest.raises(ocr.OcrError, match="closed"):
        call(**args)
