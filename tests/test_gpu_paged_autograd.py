"""What autograd knows of the paged calls: tangents and gradients that they do not
form are refused, and what they write is marked as written."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from rotatek_amd.kernels import paged_decode, paged_prefill, window_attention
from rotatek_amd.paged import append_pages
from rotatek_amd.rotary import apply_rotary, inverse_frequencies

pytestmark = pytest.mark.gpu


class Step:
    def __init__(self):
        torch.manual_seed(0)
        dt = torch.bfloat16
        self.q, self.k, self.v = (torch.randn(3, h, 64, device="cuda").to(dt) for h in (4, 2, 2))
        self.kp, self.vp = (torch.randn(6, 2, 16, 64, device="cuda").to(dt) for _ in range(2))
        self.table = torch.arange(6, dtype=torch.int32, device="cuda").view(3, 2)
        self.lens = torch.tensor([5, 17, 32], dtype=torch.int32, device="cuda")
        self.starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
        self.pos, self.freq = torch.arange(3, device="cuda"), inverse_frequencies(64)
        self.out = torch.zeros(3, 4, 64, dtype=dt, device="cuda")
        self.k_out = torch.zeros(3, 2, 64, dtype=dt, device="cuda")

    def calls(self):
        """name -> (call, names of what it reads with a gradient in mind, names of what it writes)."""
        s = self
        return {
            "rotary": (lambda: apply_rotary(s.q, s.k, s.pos, s.freq, out=(s.out, s.k_out)), "q k freq", "out k_out"),
            "append": (lambda: append_pages(s.k, s.v, s.kp, s.vp, s.table, s.lens, positions=s.pos, inv_freq=s.freq, q=s.q,
                                            q_out=s.out), "k v q freq", "kp vp out"),
            "decode": (lambda: paged_decode(s.q, s.kp, s.vp, s.table, s.lens, 2, out=s.out), "q kp vp", "out"),
            "prefill": (lambda: paged_prefill(s.q, s.starts, s.kp, s.vp, s.table, s.lens, 2, out=s.out), "q kp vp", "out"),
            "window": (lambda: window_attention(s.q.view(1, 3, 4, 64).transpose(1, 2), s.k.view(1, 3, 2, 64).transpose(1, 2),
                                                s.v.view(1, 3, 2, 64).transpose(1, 2), 2,
                                                out=s.out.view(1, 3, 4, 64).transpose(1, 2)), "q k v", "out"),
        }


CALLS = ["rotary", "append", "decode", "prefill", "window"]


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    s = Step()
    call, reads, _ = s.calls()[name]
    for x in reads.split():
        with fw.dual_level():
            plain = getattr(s, x)
            setattr(s, x, fw.make_dual(plain, torch.ones_like(plain)))
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            setattr(s, x, plain)
    call()


@pytest.mark.parametrize("name", CALLS)
def test_what_is_written_is_marked(name):
    """Autograd has to see that a tensor it saved has changed since."""
    s = Step()
    call, reads, writes = s.calls()[name]
    before = {x: getattr(s, x)._version for x in set(reads.split()) | set(writes.split()) | {"table", "lens"}}
    call()
    for x, v in before.items():
        assert (getattr(s, x)._version > v) == (x in writes.split()), x
    w = torch.ones(3, 4, 64, device="cuda", requires_grad=True)
    y = (w * s.out).sum()       # saves out
    call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_what_is_written_in_inference_mode():
    with torch.inference_mode():
        s = Step()
        for call, _, _ in s.calls().values():
            call()
    for call, _, _ in s.calls().values():       # (tensors of that mode have no count)
        call()


@pytest.mark.parametrize("name", CALLS)
def test_outputs_that_want_a_gradient_are_refused(name):
    s = Step()
    call, _, writes = s.calls()[name]
    for x in writes.split():
        plain = getattr(s, x)
        setattr(s, x, plain.detach().clone().requires_grad_())
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
        setattr(s, x, plain)
