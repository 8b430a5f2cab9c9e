"""The operators have no gradients: what would cut a graph is refused."""
import pytest

import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def calls():
    t, k = G.T(), G.K()
    make = lambda *s: t.zeros(*s, dtype=t.bfloat16, device="cuda")  # noqa: E731
    c = G.new_cache(3, 16, 2, 64, 0)[0]
    lin = dict(x=make(4, 64), w=make(32, 64), bias=make(32), mul=make(4, 32), residual=make(4, 32), out=make(4, 32))
    rows = dict(k=make(2, 2, 64), v=make(2, 2, 64))
    att = dict(q=make(2, 4, 64), out=make(2, 4, 64))
    return [(lambda **a: k.linear(G.ctx(), **a), lin), (lambda **a: c.append(slots=G.i32([0, 1]), **a), rows),
            (lambda **a: c.attention(table=G.i32([[0, 1]]), start=G.i32([0, 2]), kv_len=G.i32([2]), **a), att)]


def test_refused_where_autograd_would_follow():
    t, H = G.T(), __import__("haagenti_amd")
    for call, args in calls():
        call(**args)
        for name in args:
            asks = {**args, name: args[name].clone().requires_grad_()}
            with pytest.raises(H.HaagentiError) as e:
                call(**asks)
            assert e.value.code == H.UNSUPPORTED
            for mode in (t.no_grad, t.inference_mode):
                with mode():
                    call(**asks)
