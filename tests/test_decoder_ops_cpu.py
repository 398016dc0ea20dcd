"""Argument checks of the decoder operators that need no GPU."""
import pytest
import torch


def test_a_vector_that_has_to_be_given_is_not_made_up():
    from aesrc2020_amd.attention import _given
    t = torch.zeros(8)
    assert _given("lse", t[1:], (7,), torch.float32, t.device).data_ptr() == t.data_ptr() + 4        # a view on 4-byte boundaries will do
    for bad in (None, t, t[::2], t.double()[1:], t.view(7 + 1, 1)[1:]):
        with pytest.raises(ValueError, match="lse"):
            _given("lse", bad, (7,), torch.float32, t.device)


def test_missing_tensors_are_refused():
    from aesrc2020_amd.attention import cross_attention, cross_attention_grad
    from aesrc2020_amd.losses import vocab_crossentropy
    for f in (lambda: cross_attention(None, None, None), lambda: cross_attention_grad(None, None, None, None, None, None), lambda: vocab_crossentropy(None, None, None),
              lambda: vocab_crossentropy(torch.zeros(2, 8), torch.zeros(8, 5), None)):
        with pytest.raises(ValueError):
            f()
