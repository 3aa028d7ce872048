"""PoMStack pickled whole: as it is, and as it was before it had norms and a choice of activations.  No GPU."""
import copy
import io

import torch

from pom_b200.stack import PoMStack


def through_a_file(m):
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


def test_round_trip():
    for kw in (dict(), dict(norm=True, bias=True, activation="silu")):
        a = PoMStack(16, 2, 2, 2, **kw)
        for b in (through_a_file(a), copy.deepcopy(a)):
            assert b.activation == a.activation and len(b.norm_mix) == len(a.norm_mix)
            assert [k for k, _ in b.named_parameters()] == [k for k, _ in a.named_parameters()]
            assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


def test_a_stack_from_before_the_norms():
    old = PoMStack(16, 2, 2, 2)
    del old.__dict__["activation"], old._modules["norm_mix"], old._modules["norm_ffn"]
    new = through_a_file(old)
    assert new.activation == "gelu" and len(new.norm_mix) == len(new.norm_ffn) == 0
    h = torch.ones(1, 4, 16)
    assert new._normed(new.norm_mix, 0, h) is h
    assert list(new.state_dict()) == list(PoMStack(16, 2, 2, 2).state_dict())
