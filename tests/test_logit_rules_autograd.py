"""What autograd sees of ``logit_rules``, which has no gradient: on meta tensors, without a GPU, and on one."""
import pytest
import torch


def devices():
    return ["meta", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", devices())
def test_a_result_written_over_is_noticed(device):
    """exp keeps its result; rules on it in place make a backward pass through it wrong, so it has to refuse."""
    import torch_ggml_ops_b200 as tgo

    w = torch.zeros(2, 40, device=device, requires_grad=True)
    for out_of in (lambda e: e.detach(), lambda e: e.detach()[:1]):
        e = w.exp()
        x = out_of(e)
        before = x._version
        tgo.logit_rules(x, presence_penalty=1.0, out=x)
        assert x._version == before + 1 and e._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            e.sum().backward()
    # another tensor's memory stays what it is, and so does its version
    e = w.exp()
    y = tgo.logit_rules(e.detach(), presence_penalty=1.0)
    tgo.logit_rules(e.detach(), presence_penalty=1.0, out=y)
    assert e._version == 0 and y._version == 1
    e.sum().backward()
    with torch.no_grad():                                 # without autograd and in inference mode, too
        tgo.logit_rules(y, out=y)
    with torch.inference_mode():
        tgo.logit_rules(y, out=y)
        z = y + 0
        tgo.logit_rules(z, out=z)
    assert y._version == 3
    tgo.logit_rules(z, out=z)                             # z has no version; it can still be written


@pytest.mark.parametrize("device", devices())
def test_what_wants_a_gradient_is_refused(device):
    import torch_ggml_ops_b200 as tgo

    x = torch.zeros(2, 40, device=device)
    h, ids = torch.zeros(2, 3, dtype=torch.int64, device=device), torch.zeros(2, 1, dtype=torch.int32, device=device)
    wants = lambda *s: torch.zeros(*s, device=device, requires_grad=True)   # noqa: E731
    values = torch.zeros(2, 1, device=device)
    calls = [dict(repetition_penalty=wants(2)), dict(presence_penalty=wants(2)), dict(frequency_penalty=wants(2)), dict(bias_ids=ids, bias_values=wants(2, 1))]
    for out in (None, torch.empty_like(x)):
        for kw in calls:
            with pytest.raises(RuntimeError, match="no gradient"):
                tgo.logit_rules(x, history=h, out=out, **kw)
        with pytest.raises(RuntimeError, match="no gradient"):
            tgo.logit_rules(wants(2, 40), history=h, out=out)
    for out in (wants(2, 40), wants(2, 40) * 1):
        with pytest.raises(RuntimeError, match="no gradient"):
            tgo.logit_rules(x, history=h, out=out)
    # without autograd they are tensors like any others
    with torch.no_grad():
        leaf = wants(2, 40)
        assert tgo.logit_rules(leaf, history=h, out=leaf) is leaf
        for kw in calls:
            assert not tgo.logit_rules(leaf, history=h, **kw).requires_grad
    assert not tgo.logit_rules(x, history=h, bias_ids=ids, bias_values=values).requires_grad
