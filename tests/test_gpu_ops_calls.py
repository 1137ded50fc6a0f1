"""How the serving operators take their arguments: gradients of either mode, numbers of any kind."""
import pytest

torch = pytest.importorskip("torch")
import chatterbox_amd as cb  # noqa: E402

pytestmark = pytest.mark.gpu


def calls():
    """Each operator on (a float tensor in each place that takes one): name, tensors by name, call."""
    k, v = (torch.randn(3, 16, 2, 64, device="cuda") for _ in range(2))
    table, lens = torch.arange(3, dtype=torch.int32, device="cuda")[:, None], torch.full((3,), 9, dtype=torch.int32, device="cuda")
    kn, vn, q = (torch.randn(3, h, 64, device="cuda") for h in (2, 2, 4))
    rope = torch.randn(2, 16, 32, device="cuda")
    l, u = torch.randn(2, 3, 50, device="cuda")
    each, tok = torch.rand(3, device="cuda") + 0.5, torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    return [("attention", dict(q=q, k=k, v=v), lambda t: cb.paged_attention(t["q"], t["k"], t["v"], table, lens)),
            ("append", dict(kn=kn, vn=vn, q=q, cos=rope[0], sin=rope[1], k=k, v=v),
             lambda t: cb.paged_kv_append(t["kn"], t["vn"], t["k"], t["v"], table, lens, q=t["q"], rope=(t["cos"], t["sin"]))),
            ("logits", dict(l=l, u=u, rep=each, bias=l[:, :2]),
             lambda t: cb.process_logits(t["l"], uncond=t["u"], cfg_weight=0.5, tokens=tok, n_tokens=lens, repetition_penalty=t["rep"],
                                         bias_ids=tok[:, :2], bias_values=t["bias"]))]


def test_forward_mode_gradients_are_refused():
    """A tensor with a tangent used to come through, its tangent dropped; within a level, tensors without one are taken."""
    from torch.autograd import forward_ad as fwd
    for name, tensors, call in calls():
        want = call(tensors)
        with fwd.dual_level():
            for which in tensors:
                dual = dict(tensors)
                dual[which] = fwd.make_dual(tensors[which], torch.ones_like(tensors[which]))
                with pytest.raises(ValueError, match="forward-mode"):
                    call(dual)
                with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                    call(dual)
            assert torch.equal(call(tensors), want), name
        assert torch.equal(call(tensors), want), name


def test_reverse_mode_gradients_are_refused_where_they_are_recorded():
    for name, tensors, call in calls():
        want = call(tensors)
        for which in tensors:
            leaf = dict(tensors)
            leaf[which] = tensors[which].clone().requires_grad_()
            with pytest.raises(ValueError, match="gradients"):
                call(leaf)
            with torch.no_grad():
                assert torch.equal(call(leaf), want), (name, which)


def test_a_penalty_is_a_number_of_any_kind():
    """numpy's fp32 scalars are no Python floats; what is no number is named."""
    np = pytest.importorskip("numpy")
    l, tok, n = torch.randn(3, 50, device="cuda"), torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4), torch.full((3,), 4, dtype=torch.int32, device="cuda")
    for name, x in (("repetition_penalty", 1.25), ("frequency_penalty", 0.5), ("presence_penalty", 2.0)):
        want = cb.process_logits(l, tokens=tok, n_tokens=n, **{name: x})
        for kind in (np.float32, np.float64, np.float16):
            assert torch.equal(cb.process_logits(l, tokens=tok, n_tokens=n, **{name: kind(x)}), want)
        with pytest.raises(TypeError):
            cb.process_logits(l, tokens=tok, n_tokens=n, **{name: "1.25"})
