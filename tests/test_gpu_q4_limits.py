"""What the calls on 4-bit caches take at their limits: values, weights and gates of any size, more prompts than one
group of scratch holds, and scratch that grows."""
import pytest

from tests.test_gpu_q4 import Model, dev

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_prompt_groups_of_sequences():
    """Five sequences of 120000 cached rows: the f16 rows of four fill the scratch of one group."""
    n, lens = 120000, [3, 1, 40, 2, 130]
    m = Model([n + t for t in lens], kvc=4, seed=314)
    torch.manual_seed(314)
    for s in range(5):
        m.ctx.kv_import(0, s, torch.randn(n, 4, 256, device="cuda"), torch.randn(n, 4, 256, device="cuda"))
    qg, k, v = (dev(x) for x in m.inputs(sum(lens)))
    pos = torch.randint(0, 1 << 20, (sum(lens), 3), device="cuda", dtype=torch.int32)
    out = torch.empty(sum(lens), m.nq * 256, device="cuda")
    m.ctx.gqa_prefill_q4(0, range(5), lens, qg, k, v, out, pos=pos)
    a = 0
    for s, t in enumerate(lens):                      # one at a time: the same bits
        m.ctx.kv_truncate(0, s, n)
        one = torch.empty(t, m.nq * 256, device="cuda")
        b = slice(a, a + t)
        m.ctx.gqa_prefill_q4(0, [s], [t], qg[b], k[b], v[b], one, pos=pos[b])
        assert torch.equal(one, out[b]), s
        a += t
    m.done()
