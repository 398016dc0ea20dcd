"""Arguments of the decoder operators that only a device shows: what is missing, what lies where."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gradients_need_the_forwards_statistics():
    """lse and dloss are inputs: None is refused, a view that starts off a 16-byte boundary is taken."""
    from aesrc2020_amd.attention import cross_attention, cross_attention_grad
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(2, n, 2, 16, generator=g, device="cuda") for n in (5, 9, 9, 5))
    out, lse = cross_attention(q, k, v, return_lse=True)
    x, w = torch.randn(6, 32, generator=g, device="cuda"), torch.randn(32, 64, generator=g, device="cuda")
    lab, dl = torch.arange(6, device="cuda"), torch.rand(6, generator=g, device="cuda")
    _, zl = vocab_crossentropy(x, w, lab, return_lse=True)
    for f in (lambda: cross_attention_grad(do, q, k, v, out, None), lambda: cross_attention_grad(do, q, k, v, None, lse), lambda: cross_attention_grad(None, q, k, v, out, lse),
              lambda: vocab_crossentropy_grad(dl, x, w, lab, None), lambda: vocab_crossentropy_grad(None, x, w, lab, zl), lambda: vocab_crossentropy_grad(dl, x, w, None, zl)):
        with pytest.raises(ValueError):
            f()
    off = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)  # noqa: E731
    assert off(lse).data_ptr() % 16 == 4
    for a, b in zip(cross_attention_grad(do, q, k, v, out, off(lse)), cross_attention_grad(do, q, k, v, out, lse)):
        assert torch.equal(a, b)
    for a, b in zip(vocab_crossentropy_grad(off(dl), x, w, lab, off(zl))[:2], vocab_crossentropy_grad(dl, x, w, lab, zl)[:2]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("Tq", [3, 90])
def test_results_go_into_any_contiguous_buffer(Tq):
    """An axis of length 1 may have any stride in a contiguous tensor (a transposed or sliced buffer)."""
    from aesrc2020_amd.attention import EncoderCache8, cross_attention, cross_attention_grad
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, do = (torch.randn(1, n, 1, 64, generator=g, device="cuda") for n in (Tq, 70, 70, Tq))
    cache = EncoderCache8(1, 70, 1, 64)
    cache.store(k, v)
    want, lse = cross_attention(q, k, v, return_lse=True)
    held = cache.attend(q)
    grads = cross_attention_grad(do, q, k, v, want, lse)
    for make in (lambda n: torch.empty(1, n, 64, 1, device="cuda").transpose(2, 3), lambda n: torch.empty(1 * n * 64, device="cuda").as_strided((1, n, 1, 64), (3, 64, 7, 1))):
        out = make(Tq)
        assert out.is_contiguous() and cross_attention(q, k, v, out=out) is out and torch.equal(out, want)
        assert cache.attend(q, out=out) is out and torch.equal(out, held)
        got = cross_attention_grad(do, q, k, v, out.copy_(want), lse, dq=make(Tq), dk=make(70), dv=make(70))
        assert all(torch.equal(a, b) for a, b in zip(got, grads))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_the_layer_is_the_calls_in_every_type(dt):
    """CrossAttention over rows of any of the three types, shared key heads, padded on both sides: bit for bit what the functions give."""
    from aesrc2020_amd.attention import cross_attention, cross_attention_grad
    from aesrc2020_amd.engine import ParamStore, store_scope
    from aesrc2020_amd.layers import CrossAttention
    B, Lq, Lk, H, heads, kv = 3, 20, 50, 96, 6, 2
    g = torch.Generator(device="cuda").manual_seed(4)
    q, dy = (torch.randn(B * Lq, H, generator=g, device="cuda").to(dt) for _ in range(2))
    k, v = (torch.randn(B * Lk, H // heads * kv, generator=g, device="cuda").to(dt) for _ in range(2))
    kl, ql = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ((50, 0, 33), (20, 7, 0)))
    with store_scope(ParamStore(seed=0)):
        layer = CrossAttention(H, heads, kv, name="att")
    y = layer.forward(q, k, v, B, Lq, Lk, kl, ql)
    grads = layer.backward(dy)
    view = lambda t, n: t.view(B, -1, n, H // heads)  # noqa: E731
    out, lse = cross_attention(view(q, heads), view(k, kv), view(v, kv), kl, ql, return_lse=True)
    want = cross_attention_grad(view(dy, heads), view(q, heads), view(k, kv), view(v, kv), out, lse, kl, ql)
    assert y.dtype == dt and torch.equal(y, out.view(B * Lq, H))
    for a, b in zip(grads, want):
        assert a.dtype == dt and torch.equal(a, b.view(a.shape)) and (a != 0).any()
