"""The decoder operators captured into HIP graphs, in the forms that larger calls take: two graphs alive at once, replayed in turn with eager work between,
every replay against the eager result on the inputs of the moment."""
import pytest
import torch

from tests.test_gpu_attention import DT
from tests.test_gpu_attention import make as attention_inputs
from tests.test_gpu_vocab_ce import make as loss_inputs

pytestmark = pytest.mark.gpu


def replay_all(builds, change):
    """builds: calls -> tensors.  Captures each, then four rounds of change(i), the replays, the eager calls."""
    for f in builds:
        f()
    torch.cuda.synchronize()
    graphs = []
    for f in builds:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = f()
        graphs.append((g, held))
    for i in range(4):
        change(i)
        for g, _ in graphs:
            g.replay()
        eager = [f() for f in builds]
        torch.cuda.synchronize()
        for (_, held), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(held, want) if a is not None), i


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", [(2000, 256, 700), (1100, 637, 4001), (8200, 64, 20011)])
def test_vocabulary_loss_and_gradients(R, D, V, dt):
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = loss_inputs(R, D, V, DT[dt], seed=1)
    y = loss_inputs(R, D, V, DT[dt], seed=2)[0]

    def step(t):
        loss, lse = vocab_crossentropy(t, w, lab, b, return_lse=True)
        return (loss, lse) + vocab_crossentropy_grad(dl, t, w, lab, lse, b)

    def change(i):
        n = loss_inputs(R, D, V, DT[dt], seed=10 + i)
        x.copy_(n[0] * 4 ** i); w.copy_(n[1]); lab.copy_((n[2] + i).clamp_max(V)); dl.copy_(n[4] * 8.0 ** i)
    replay_all([lambda: step(x), lambda: step(y)], change)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shape", [(2, 70, 39, 4, 2, 64), (1, 130, 200, 4, 2, 128), (2, 300, 700, 4, 2, 64), (16, 500, 301, 8, 8, 40), (1, 9, 5000, 2, 1, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_attention_and_gradients(shape, dt):
    from aesrc2020_amd.attention import cross_attention, cross_attention_grad
    q, k, v, g = attention_inputs(*shape, DT[dt], seed=1)
    kl = torch.full((shape[0],), shape[2], dtype=torch.int32, device="cuda")

    def step(a, c):
        out, lse = cross_attention(q, a, c, k_lens=kl, return_lse=True)
        return (out, lse) + cross_attention_grad(g, q, a, c, out, lse, k_lens=kl)

    def change(i):
        n = attention_inputs(*shape, DT[dt], seed=20 + i)
        for t, s, f in zip((q, k, v, g), n, (1, 1, 1, 10.0 ** -i)):
            t.copy_(s * f)
        kl.fill_(max(0, shape[2] - 13 * i))
    replay_all([lambda: step(k, v), lambda: step(v, k)], change)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("Tq,Tk", [(1, 189), (5, 3000)])
def test_cache_written_and_read(Tq, Tk, dt):
    """A graph that stores and attends, beside one that attends only to the same cache."""
    from aesrc2020_amd.attention import EncoderCache8
    q, k, v, _ = attention_inputs(3, Tq, Tk, 4, 2, 64, DT[dt], seed=1)
    n = torch.tensor([Tk, Tk // 2, 1], dtype=torch.int32, device="cuda")
    c = EncoderCache8(3, Tk, 2, 64)

    def both():
        c.store(k, v, n)
        return (c.attend(q), c.k8.view(torch.uint8).clone(), c.v_scale.clone())

    def change(i):
        m = attention_inputs(3, Tq, Tk, 4, 2, 64, DT[dt], seed=30 + i)
        for t, s in zip((q, k, v), m):
            t.copy_(s * 4.0 ** i)
        n.copy_(torch.tensor([Tk - i, i * 64, Tk // 3], dtype=torch.int32))
    replay_all([both, lambda: (c.attend(q),)], change)
