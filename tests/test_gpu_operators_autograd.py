"""The operators among PyTorch's autograd: saved-tensor hooks, checkpointing, what changes between
the passes."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tests.test_gpu_operators import BF, SF, Batch, _padded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from temporal_random_walk import operators
    return operators


NAMES = ("out", "d_q", "d_k", "d_v", "d_table")


class Case:
    """Walks with every term of a score, and the gradients of one pass over them."""

    def __init__(self, ops, dtype, padded, lens):
        b = Batch(lens, heads=4, kv_heads=2, dtype=dtype, softcap=20.0, slopes=True, times=True,
                  buckets=ops.distance_buckets(6, 9, device="cpu"), num_buckets=6)
        self.ops, self.b = ops, b
        self.given = [b.q, b.k, b.v]
        self.d_out = b.d_out
        self.terms = b.terms()
        if padded:
            length = max(lens)
            self.given = [_padded(x, lens, length) for x in self.given]
            self.d_out = _padded(b.d_out, lens, length)
            times = _padded(b.q_times, lens, length).cuda()
            self.terms.update(times=times, k_times=times)
            self.mask = ops.WalkMask.padded(torch.tensor(lens).cuda(), length)
        else:
            self.mask = b.mask(ops)

    def leaves(self):
        return [x.cuda().requires_grad_() for x in self.given + [self.b.table]]

    def attention(self, q, k, v, table):
        return self.ops.walk_attention(q, k, v, self.mask, **{**self.terms, "bias_table": table})

    def grads(self, out, leaves):
        return dict(zip(NAMES, (out.detach(),
                                *torch.autograd.grad(out, leaves, self.d_out.cuda()))))

    def run(self):
        leaves = self.leaves()
        return self.grads(self.attention(*leaves), leaves)


# short walks (a wave each), and walks that take tiles
CASES = [(dtype, padded, lens) for dtype in (BF, SF) for padded in (False, True)
         for lens in ([20, 1, 33, 40], [130, 7, 0, 300])]


@pytest.mark.parametrize("dtype,padded,lens", CASES)
def test_checkpointing(ops, dtype, padded, lens):
    """Recomputed in the backward pass, with nothing kept between the passes: bit for bit the same."""
    case = Case(ops, dtype, padded, lens)
    want = case.run()
    leaves = case.leaves()

    def block(q, k, v, table):  # inputs that only the block's own history holds
        return case.attention(q * 1, k * 1, v * 1, table * 1) * 1

    out = checkpoint(block, *leaves, use_reentrant=False)
    held = [torch.randn(1 << 20, device="cuda") for _ in range(8)]  # takes the memory that was freed
    got = case.grads(out, leaves)
    assert len(held) == 8
    for name in want:
        assert torch.equal(torch.nan_to_num(got[name]), torch.nan_to_num(want[name])), name


@pytest.mark.parametrize("dtype,padded,lens", CASES)
def test_saved_tensor_hooks(ops, dtype, padded, lens):
    """The backward pass reads what the hooks give back and not what was packed: copies with other
    strides, while the packed ones are overwritten."""
    case = Case(ops, dtype, padded, lens)
    want = case.run()
    leaves = [x.detach().clone().requires_grad_() for x in case.leaves()]
    packed = []

    def pack(x):
        wide = x.new_zeros(x.shape[:-1] + (x.shape[-1] + 3,))[..., 3:]
        packed.append(x.detach())
        return wide.copy_(x.detach())

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda x: x):
        out = case.attention(*leaves)
        first = out.detach().clone()
    with torch.no_grad():
        for x in packed:
            x.fill_(1 if x.dtype == torch.int32 else float("nan"))
    got = case.grads(out, leaves)
    got["out"] = first
    for name in want:
        assert torch.equal(torch.nan_to_num(got[name]), torch.nan_to_num(want[name])), name


def test_saved_on_the_host(ops):
    case = Case(ops, BF, False, [130, 7, 0, 300])
    want = case.run()
    leaves = case.leaves()
    with torch.autograd.graph.save_on_cpu():
        out = case.attention(*leaves)
    got = case.grads(out, leaves)
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_bias_under_hooks(ops):
    table = torch.randn(3, 5, device="cuda", requires_grad=True)
    ids = ops.distance_buckets(5, 7)
    d = torch.randn(3, 20, 30, device="cuda")
    (want,) = torch.autograd.grad(ops.relative_bias(table, ids, 20, 30), table, d)
    with torch.autograd.graph.save_on_cpu():
        out = ops.relative_bias(table, ids, 20, 30)
    (got,) = torch.autograd.grad(out, table, d)
    assert torch.equal(got, want)


@pytest.mark.parametrize("other", ["device", "type", "shape"])
def test_hooks_that_give_back_something_else(ops, other):
    """Refused on the host: nothing is read that is not there."""
    change = {"device": lambda x: x.cpu(), "type": lambda x: x.double(),
              "shape": lambda x: x.unsqueeze(0)}[other]
    case = Case(ops, SF, False, [20, 3])
    leaves = case.leaves()
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x.detach(), change):
        out = case.attention(*leaves)
        bias = ops.relative_bias(leaves[3], case.terms["buckets"], 6, 6)
    for x in (out, bias):
        with pytest.raises(RuntimeError, match="came back from its hook"):
            x.backward(torch.zeros_like(x))


@pytest.mark.parametrize("lens", [[20, 3], [130, 200]])
@pytest.mark.parametrize("name", ["times", "k_times", "slopes", "buckets"])
def test_terms_changed_between_the_passes(ops, name, lens):
    """The backward pass works the scores out again: a term that has changed is an error."""
    case = Case(ops, SF, False, lens)
    want = case.run()
    case.terms["k_times"] = case.terms["times"].clone()
    leaves = case.leaves()
    out = case.attention(*leaves)
    case.terms[name].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        case.grads(out, leaves)
    case.terms[name].sub_(1)
    out = case.attention(*leaves)
    got = case.grads(out, leaves)
    for x in want:
        assert torch.allclose(got[x], want[x], rtol=0, atol=1e-3), x


def test_buckets_changed_between_the_passes_of_the_bias(ops):
    table = torch.randn(3, 5, device="cuda", requires_grad=True)
    ids = ops.distance_buckets(5, 7)
    out = ops.relative_bias(table, ids, 20, 30)
    ids.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def _event(requires_grad=False, dtype=SF, times=False):
    x = dict(q=torch.randn(3, 4, 64, dtype=dtype, device="cuda", requires_grad=requires_grad),
             k=torch.randn(3, 2, 64, dtype=dtype, device="cuda"),
             v=torch.randn(3, 2, 64, dtype=dtype, device="cuda"),
             k_cache=torch.randn(3, 16, 2, 64, dtype=dtype, device="cuda"),
             v_cache=torch.randn(3, 16, 2, 64, dtype=dtype, device="cuda"),
             lens=torch.tensor([0, 5, -1]).cuda())
    if times:
        x.update(slopes=torch.ones(4, device="cuda"), times=torch.ones(3, device="cuda"),
                 k_times=torch.zeros(3, 16, device="cuda"))
    return x


@pytest.mark.parametrize("name", ["k_cache", "v_cache", "k_times"])
def test_a_step_changes_its_caches(ops, name):
    """What saved a cache before a step learns that the step wrote to it."""
    event = _event(times=True)
    weight = torch.ones((), device="cuda", requires_grad=True)
    product = weight * event[name]
    ops.walk_attention_step(**event)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    product = weight * event["q"]  # what it only reads is as it was
    ops.walk_attention_step(**event)
    product.sum().backward()


def test_a_step_in_inference_mode(ops):
    with torch.inference_mode():
        event = _event(times=True)
        want = ops.walk_attention_step(**event)
    with torch.no_grad():  # caches that track no versions
        assert torch.equal(ops.walk_attention_step(**event), want)


def test_a_step_has_no_gradient(ops):
    """It says so where one is asked for."""
    event = _event(requires_grad=True)
    out = ops.walk_attention_step(**event)
    with pytest.raises(RuntimeError, match="walk_attention_step has no gradient"):
        out.sum().backward()
    for name in ("k", "v", "k_cache", "v_cache", "bias_table"):
        event = _event()
        event.update(bias_table=torch.randn(4, 3, device="cuda"),
                     buckets=torch.tensor([0, 1, 2], dtype=torch.int32).cuda())
        event[name].requires_grad_()
        with pytest.raises(RuntimeError, match="walk_attention_step has no gradient"):
            ops.walk_attention_step(**event).sum().backward()
    event = _event(requires_grad=True)  # also where the input is reached another way
    loss = ops.walk_attention_step(**event).sum() + event["q"].sum()
    with pytest.raises(RuntimeError, match="walk_attention_step has no gradient"):
        torch.autograd.grad(loss, event["q"])
    with torch.no_grad():
        assert not ops.walk_attention_step(**_event(requires_grad=True)).requires_grad
    assert not ops.walk_attention_step(**_event()).requires_grad


def test_a_step_has_no_forward_derivative(ops):
    import torch.autograd.forward_ad as fwad
    event = _event()
    with fwad.dual_level():
        event["q"] = fwad.make_dual(event["q"], torch.ones_like(event["q"]))
        with pytest.raises(RuntimeError, match="walk_attention_step has no gradient"):
            ops.walk_attention_step(**event)


def test_terms_of_the_inference_mode(ops):
    """Constant terms that were made there serve a training pass too."""
    case = Case(ops, SF, False, [20, 3])
    want = case.run()
    with torch.inference_mode():
        case.terms.update({name: x.clone() for name, x in case.terms.items()
                           if isinstance(x, torch.Tensor) and name != "bias_table"})
    got = case.run()
    for name in want:
        assert torch.equal(got[name], want[name]), name
    table = torch.randn(3, 6, device="cuda", requires_grad=True)
    ops.relative_bias(table, case.terms["buckets"], 20, 30).sum().backward()
    assert table.grad is not None
