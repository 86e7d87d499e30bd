"""GPU: attention of several new tokens over sequences that lie in one large page, whose rows pass 4 GiB."""
import ctypes

import numpy as np
import pytest
import torch

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from prompt_call import many_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,rows,dim,shift", [("bf16", "bf16", 256, 24), ("f16", "f16", 128, 25), ("int8", "bf16", 256, 25)])
@pytest.mark.parametrize("new,group", [(600, 16), (2, 4)])
def test_a_page_past_4_gib(kind, rows, dim, shift, new, group):
    """A page of 2^24 or 2^25 tokens, 8 GiB; the last `new` of a sequence that ends near its end."""
    pk.call("pk_gpu_init", 0)
    page, pages, window = 1 << shift, 1, 200
    length = page - 70
    assert many_rows(kind, rows, 1, group, 1, new, page, window) == (new > 2)
    tt = do.torch_type(kind)
    k, v = (torch.zeros((pages * page * dim,), dtype=tt, device="cuda:0") for _ in range(2))
    scales = [torch.zeros((pages * page,), device="cuda:0") for _ in range(2)] if kind == "int8" else [None, None]
    at = lambda t: None if t is None else t.data_ptr()
    c = pk.KvCache(k.data_ptr(), v.data_ptr(), at(scales[0]), at(scales[1]), do.KINDS[kind], pages, page, 1, dim)
    n = new + window                                      # the tokens that are seen
    rt = do.torch_type(rows)
    x, y = (torch.randn((n, dim), device="cuda:0").to(rt) for _ in range(2))
    q = torch.randn((new, group * dim), device="cuda:0").to(rt)
    out = torch.zeros_like(q)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda:0")
    slots = ints(np.arange(length - n, length))
    pk.call("pk_gpu_kv_write_dev", do.ref(c), do.FLOATS[rows], x.data_ptr(), dim, y.data_ptr(), dim, slots.data_ptr(), n, do.stream())
    table, lens, starts = ints([[0]]), ints([length]), ints([0, new])
    rules = pk.AttentionRules(dim ** -0.5, 0.0, None, window, None, None)
    floats = pk.load().pk_gpu_prompt_attention_ws_floats(do.ref(c), 1, new, group, new, page, window)
    ws = torch.empty((floats + 4,), device="cuda:0")
    pk.call("pk_gpu_prompt_attention_dev", do.ref(c), do.FLOATS[rows], q.data_ptr(), group * dim, group, table.data_ptr(), 1,
            lens.data_ptr(), starts.data_ptr(), 1, new, new, page, ctypes.byref(rules), out.data_ptr(), group * dim, None,
            ws.data_ptr(), floats, do.stream())
    back = [torch.zeros((n, dim), device="cuda:0") for _ in range(2)]
    pk.call("pk_gpu_kv_read_dev", do.ref(c), pk.F32, slots.data_ptr(), n, back[0].data_ptr(), dim, back[1].data_ptr(), dim, do.stream())
    torch.cuda.synchronize()

    class Rows:          # what the cache's rows stand for, by token
        heads, page, pages = 1, 1, n
    held = Rows()
    held.dim, held.kind = dim, kind
    held.rows = {"k": do.values(back[0]).reshape(n, 1, dim), "v": do.values(back[1]).reshape(n, 1, dim)}.__getitem__
    want = mo.Ruled(held, do.values(q).reshape(new, group, dim), np.arange(n)[None], [n], [0, new], new, n, dim ** -0.5, window=window)
    err = np.abs(do.values(out).reshape(new, group, dim) - want.out)
    assert np.all(err <= want.bound(kind, rows, mo.half_of_weights(kind, rows, new > 2)))
