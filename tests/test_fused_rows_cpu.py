"""Which modules' decode steps apply_patch(fused_qk=True) sends through qk_norm_rope: only those whose norms are plain
RMS norms that nobody watches or replaces.  The kernel call is recorded, not made (no GPU needed)."""
import pytest
import torch

HD = 64


class RMSNorm(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(HD))
        self.variance_epsilon = 1e-6

    def forward(self, x):
        return self.weight * x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.variance_epsilon)


class Attention(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.q_norm, self.k_norm = RMSNorm(), RMSNorm()


@pytest.fixture
def fused(monkeypatch):
    from tritiercache_b200.integration import patch_model
    calls = []
    monkeypatch.setattr(patch_model._C, "qk_norm_rope", lambda *a, **kw: calls.append(kw))

    def run(module):
        del calls[:]
        z = lambda h: torch.zeros((1, 1, h, HD))  # noqa: E731
        c = torch.zeros((1, 1, HD))
        rows = patch_model._fused_rows(module, z(4), z(2), z(2), c, c, torch.device("cpu"))
        assert (rows is not None) == bool(calls)
        return rows is not None
    return run


def test_plain_norms_are_fused(fused):
    assert fused(Attention())
    assert fused(torch.nn.Module())  # no norms at all


@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
@pytest.mark.parametrize("watch", ["forward_hook", "pre_hook", "backward_hook", "backward_pre_hook", "forward"])
def test_norms_that_are_watched_or_replaced_run_themselves(fused, which, watch):
    m = Attention()
    n = getattr(m, which)
    handle = None
    if watch == "forward_hook":
        handle = n.register_forward_hook(lambda *a: None)
    elif watch == "pre_hook":
        handle = n.register_forward_pre_hook(lambda *a: None)
    elif watch == "backward_hook":
        handle = n.register_full_backward_hook(lambda *a: None)
    elif watch == "backward_pre_hook":
        handle = n.register_full_backward_pre_hook(lambda *a: None)
    else:
        n.forward = lambda x: 2 * x
    assert not fused(m)
    if handle is not None:
        handle.remove()
        assert fused(m)


def test_hooks_on_every_module_count_too(fused):
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        assert not fused(Attention())
    finally:
        handle.remove()
    assert fused(Attention())
