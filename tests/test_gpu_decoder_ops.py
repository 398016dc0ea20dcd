"""The attention-decoder operators as Layers, and a run of them together: projections (Dense), cross attention to padded encoder rows, the vocabulary
cross entropy from the last hidden rows, the whole backward into a ParamStore's gradient buffer, one Adam step, and decoding with the 8-bit cache."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _net(B, Lq, Lk, H, heads, kv_heads, V, seed=0):
    from aesrc2020_amd.engine import ParamStore, store_scope
    from aesrc2020_amd.layers import CrossAttention, Dense
    from aesrc2020_amd.losses import VocabCrossentropy
    store = ParamStore(seed=seed)
    kw = H // heads * kv_heads
    with store_scope(store):
        L = dict(q=Dense(H, H, name="q"), k=Dense(H, kw, name="k"), v=Dense(H, kw, name="v"), att=CrossAttention(H, heads, kv_heads, name="att"), pred=Dense(H, V, name="pred"))
    store.finalize()
    store.set_adam(1e-3)
    L["loss"] = VocabCrossentropy(store.bufs, "vce", L["pred"])
    return store, L


def _step(store, L, tok, enc, B, Lq, Lk, k_lens, q_lens, labels, dloss):
    store.zero_grads()
    q, k, v = L["q"].forward(tok), L["k"].forward(enc), L["v"].forward(enc)
    y = L["att"].forward(q, k, v, B, Lq, Lk, k_lens, q_lens)
    loss = L["loss"].forward(y, labels)
    dq, dk, dv = L["att"].backward(L["loss"].backward(dloss))
    L["q"].backward(dq)
    L["k"].backward(dk)
    L["v"].backward(dv)
    return loss


def _reference(store, tok, enc, B, Lq, Lk, heads, kv_heads, k_lens, q_lens, labels, dloss):
    """float64 autograd over the same weights -> (loss, {name: gradient})"""
    P = {r.name: r.w.detach().double().clone().requires_grad_() for r in store.refs}
    dense = lambda n, x: x @ P[n + "/kernel"] + P[n + "/bias"]  # noqa: E731
    D = tok.shape[1] // heads
    q = dense("q", tok.double()).view(B, Lq, heads, D).transpose(1, 2)
    k, v = (dense(n, enc.double()).view(B, Lk, kv_heads, D).transpose(1, 2).repeat_interleave(heads // kv_heads, 1) for n in "kv")
    s = (q @ k.mT) / math.sqrt(D)
    s = s.masked_fill(torch.arange(Lk, device="cuda").view(1, 1, 1, Lk) >= k_lens.view(B, 1, 1, 1), -math.inf)
    y = (torch.softmax(s, -1) @ v).transpose(1, 2)
    y = y * (torch.arange(Lq, device="cuda").view(1, Lq, 1, 1) < q_lens.view(B, 1, 1, 1))
    z = torch.log_softmax(dense("pred", y.reshape(B * Lq, -1)), 1)
    loss = torch.where(labels >= 0, -z.gather(1, labels.long().clamp_min(0)[:, None])[:, 0], torch.zeros_like(z[:, 0]))
    return loss.detach(), dict(zip(P, torch.autograd.grad(loss, list(P.values()), dloss.double())))


def _inputs(B, Lq, Lk, H, V, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tok, enc = (torch.randn(n, H, generator=g, device="cuda") for n in (B * Lq, B * Lk))
    k_lens = torch.randint(1, Lk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    q_lens = torch.randint(1, Lq + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    labels = torch.randint(0, V, (B, Lq), generator=g, device="cuda", dtype=torch.int32)
    labels[torch.arange(Lq, device="cuda")[None] >= q_lens[:, None]] = -1
    dloss = torch.full((B * Lq,), 1.0 / float(q_lens.sum()), device="cuda")
    return tok, enc, k_lens, q_lens, labels.view(-1), dloss


@pytest.mark.parametrize("B,Lq,Lk,H,heads,kv_heads,V", [(4, 18, 39, 64, 4, 4, 50), (3, 72, 100, 256, 8, 2, 1000)])
def test_training_step_of_the_three_together(B, Lq, Lk, H, heads, kv_heads, V):
    """fp32 all through (the Dense layers in their fp32 mode): every difference is fp32 rounding.  A Dense of H products carries about H^0.5 2^-24 of its
    terms' size, three of them and two attention products in a row stay below 2^-24 * 64 * sqrt(H) of a tensor's norm."""
    store, L = _net(B, Lq, Lk, H, heads, kv_heads, V)
    x = _inputs(B, Lq, Lk, H, V)
    want, grads = _reference(store, x[0], x[1], B, Lq, Lk, heads, kv_heads, *x[2:])
    loss = _step(store, L, x[0], x[1], B, Lq, Lk, *x[2:])
    lim = 2.0 ** -24 * 64 * math.sqrt(H)
    assert torch.linalg.norm(loss.double() - want) <= lim * torch.linalg.norm(want)
    # the sum of a bias gradient of the keys is 0 by the softmax's invariance: its rounding is measured against the terms, not the sum
    scale = max(float(torch.linalg.norm(g)) for g in grads.values())
    for r in store.refs:
        g = grads[r.name]
        assert torch.linalg.norm(r.g.double() - g) <= lim * max(float(torch.linalg.norm(g)), 1e-2 * scale), r.name


def test_training_step_captured_and_replayed():
    B, Lq, Lk, H, heads, V = 3, 20, 45, 64, 4, 70
    store, L = _net(B, Lq, Lk, H, heads, heads, V)
    x = list(_inputs(B, Lq, Lk, H, V))
    for _ in range(2):
        _step(store, L, x[0], x[1], B, Lq, Lk, *x[2:])
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        loss = _step(store, L, x[0], x[1], B, Lq, Lk, *x[2:])
    for i in range(3):
        for a, b in zip(x, _inputs(B, Lq, Lk, H, V, seed=10 + i)):
            a.copy_(b)
        gr.replay()
        got, gg = loss.clone(), store.grads.clone()
        _step(store, L, x[0], x[1], B, Lq, Lk, *x[2:])
        torch.cuda.synchronize()
        assert torch.equal(got, L["loss"].loss) and torch.equal(gg, store.grads)


def test_gradients_accumulate_and_adam_takes_them():
    """Two backward passes into the store are twice one; an Adam step moves every weight that has a gradient."""
    B, Lq, Lk, H, heads, V = 2, 10, 30, 64, 4, 40
    store, L = _net(B, Lq, Lk, H, heads, heads, V)
    x = _inputs(B, Lq, Lk, H, V)
    _step(store, L, x[0], x[1], B, Lq, Lk, *x[2:])
    one = L["pred"].kernel.g.clone()
    L["loss"].backward(x[-1])
    assert torch.equal(L["pred"].kernel.g, one + one)
    before = store.params.clone()
    store.adam_step()
    moved = (store.params != before)[:store.n]
    assert moved.view(-1)[store.refs[0].offset:store.refs[0].offset + store.refs[0].size].any() and torch.isfinite(store.params).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_decoding_with_the_cache_agrees_with_attention_over_its_values(dt):
    """Tokens one at a time over the 8-bit cache = the many-row kernel over the values that the cache holds."""
    from aesrc2020_amd.attention import EncoderCache8, cross_attention
    g = torch.Generator(device="cuda").manual_seed(3)
    B, T, Tk, Hq, H, D = 3, 40, 700, 8, 4, 64
    q = torch.randn(B, T, Hq, D, generator=g, device="cuda").to(dt)
    k, v = (torch.randn(B, Tk, H, D, generator=g, device="cuda").to(dt) for _ in range(2))
    lens = torch.tensor([700, 333, 1], dtype=torch.int32, device="cuda")
    c = EncoderCache8(B, Tk, H, D)
    c.store(k, v, lens)
    held = [(x.float() * s.repeat_interleave(64, 2)[..., None])[:, :, :Tk].transpose(1, 2).contiguous() for x, s in ((c.k8, c.k_scale), (c.v8, c.v_scale))]
    want = cross_attention(q.float(), held[0], held[1], k_lens=lens)
    got = torch.cat([c.attend(q[:, t:t + 1]) for t in range(T)], 1)
    # probabilities and results rounded to the type (half a step each of sum p |v| and of the result), fp32 sums
    u = torch.finfo(dt).eps / 2
    lim = (2.1 * u + 2.0 ** -15) * held[1].abs().amax((1, 3)).repeat_interleave(Hq // H, 1)[:, None, :, None]
    assert ((got.float() - want).abs() <= lim).all()


def test_two_streams_at_once():
    """Calls on two streams at the same time: each allocates its own workspace."""
    from aesrc2020_amd.attention import cross_attention, cross_attention_grad
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    g = torch.Generator(device="cuda").manual_seed(5)
    sets = []
    for i in range(2):
        q, k, v, do = (torch.randn(2, n, 4, 64, generator=g, device="cuda").to(torch.bfloat16) for n in (50, 3000, 3000, 50))
        x, w = torch.randn(500, 128, generator=g, device="cuda").half(), (torch.randn(128, 3001, generator=g, device="cuda") * 0.1).half()
        lab = torch.randint(0, 3001, (500,), generator=g, device="cuda")
        sets.append((q, k, v, do, x, w, lab, torch.full((500,), 0.01, device="cuda")))

    def run(q, k, v, do, x, w, lab, dl):
        o, l = cross_attention(q, k, v, return_lse=True)
        loss, lse = vocab_crossentropy(x, w, lab, return_lse=True)
        return (o, l, loss) + cross_attention_grad(do, q, k, v, o, l) + vocab_crossentropy_grad(dl, x, w, lab, lse)[:2]

    alone = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        both = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                both.append(run(*s))
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
