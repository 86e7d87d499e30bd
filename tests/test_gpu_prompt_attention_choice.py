"""GPU: which kernel a call of the attention with rules takes, read from a captured call, and that the rule by
which the other tests choose their bounds says the same."""
import ctypes
import re

import numpy as np
import pytest
import torch

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from prompt_call import prompt, sides
from test_gpu_prompt_attention import CASES, rules_of
from test_gpu_prompt_attention_many import PAIRINGS, TWO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


class Dim3(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint) for n in "xyz"]


class NodeParams(ctypes.Structure):
    _fields_ = [("block", Dim3), ("extra", ctypes.c_void_p), ("func", ctypes.c_void_p), ("grid", Dim3),
                ("params", ctypes.c_void_p), ("lds", ctypes.c_uint)]


def kernels(c):
    """Names of the kernels that the call launches."""
    hip = ctypes.CDLL("libamdhip64.so")
    hip.hipKernelNameRefByPtr.restype = ctypes.c_char_p
    g, s = torch.cuda.CUDAGraph(keep_graph=True), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        c.enqueue(s.cuda_stream)
    graph, n = ctypes.c_void_p(g.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(graph, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(graph, nodes, ctypes.byref(n)) == 0
    got = []
    for node in nodes:
        p = NodeParams()
        assert hip.hipGraphKernelNodeGetParams(ctypes.c_void_p(node), ctypes.byref(p)) == 0
        got.append(hip.hipKernelNameRefByPtr(ctypes.c_void_p(p.func), None).decode())
    return got


def taken(c):
    """The kernel of few rows, or the one of many and its sides; of the call's types and head size."""
    got = [k for k in kernels(c) if "paged_join" not in k]
    assert len(got) == 1
    name, cache, rows, dim, how = re.search(r"(paged|prompt)_attentionILi(\d)ELi(\d)ELi(\d+)EL([bi]\d)E", got[0]).groups()
    assert (int(cache), int(rows), int(dim)) == (mo.KINDS[c.cache.kind], do.FLOATS[c.rows], c.cache.dim)
    assert how in (("b1",) if name == "paged" else ("i1", "i2"))
    return ("few",) if name == "paged" else ("many", int(how[1]))


@pytest.mark.parametrize("kind,rows,kv,group,dim,page,new,lens,how", CASES)
def test_cases_of_all_kinds(kind, rows, kv, group, dim, page, new, lens, how):
    c = prompt(np.random.default_rng(0), kind, rows, kv, group, dim, page, new, lens, tail=3, **rules_of(how, kv * group))
    assert taken(c) == (("many", sides(c)) if c.many() else ("few",))


@pytest.mark.parametrize("kind,rows", PAIRINGS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv,group,new,lens,how", [
    (12, 3, [70, 0, 33, 129], [70, 40, 150, 131], {}), (4, 4, [11] * 5, [800] * 5, {}), (8, 1, [900], [900], {}),
    (32, 2, [200] * 3, [1000, 300, 200], {}), (16, 4, [700], [800], dict(docs=100)), (8, 4, [5] * 40, [900] * 40, {}),
])
def test_pairings(kind, rows, dim, kv, group, new, lens, how):
    c = prompt(np.random.default_rng(0), kind, rows, kv, group, dim, 64, new, lens, **rules_of(how, kv * group))
    assert taken(c) == (("many", sides(c)) if c.many() else ("few",))


@pytest.mark.parametrize("kind,rows,dim", TWO)
def test_two_sides(kind, rows, dim):
    for kv, new, lens, how in ((11, [70, 0, 33, 129], [470, 40, 450, 431], {}), (33, [360], [459], dict(window=1))):
        c = prompt(np.random.default_rng(0), kind, rows, kv, 3 if kv == 11 else 2, dim, 16, new, lens, tail=5, **how)
        assert taken(c) == ("many", 2)


@pytest.mark.parametrize("new,first,rows,want", [
    # 16 heads over 4 of 64: tiles of 128 rows at the limits of one round of workgroups, and with documents of two
    (4096, False, "bf16", 2), (4097, False, "bf16", 1), (4097, True, "bf16", 2), (8192, True, "bf16", 2), (8193, True, "bf16", 1),
    (4096, True, "f32", 2), (4097, True, "f32", 1)])
def test_limits_of_two_sides(new, first, rows, want):
    c = prompt(np.random.default_rng(0), "bf16", rows, 4, 4, 64, 64, [new], [new], first=(lambda b, p: p // 300 * 300) if first else None)
    assert taken(c) == ("many", want) and sides(c) == want
