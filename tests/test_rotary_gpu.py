"""Rotary positions against products of complex numbers in 64 bits, and their gradients."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import rotary_ref
from tokamax_b200 import rotary

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half a step of f16's subnormals


def _rows(b, heads, t, d, dtype, seed, heads_first=True):
  g = torch.Generator(device=DEV).manual_seed(seed)
  if heads_first:
    return torch.randn(b, heads, t, d, generator=g, device=DEV).to(dtype)
  return torch.randn(b, t, heads, d, generator=g, device=DEV).to(dtype).transpose(1, 2)


def _check(got, x, positions, freq, **kw):
  """An angle is rounded to 24 bits of a half turn (pi 2^-25), sine and cosine to 2 units in the last place (2^-23), both times the
  factor (2^-24), two products and their sum (2^-24 each): below 2^-21 of |x0| + |x1| in all.  Then the rounding to the type."""
  want, size = rotary_ref.rotate(x, positions, freq, **kw)
  assert got.dtype == x.dtype and got.shape == x.shape
  before = 2.0 ** -21 * size
  bound = before + (ROUNDOFF[x.dtype] * (want.abs() + before) + LEAST[x.dtype]) * (size > 0)
  err = (got.cpu().double() - want).abs()
  assert (err <= bound).all(), float((err - bound).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,dim", [(8, 2), (8, 8), (64, 64), (80, 32), (80, 40), (80, 20), (96, 96), (128, 128), (128, 32), (160, 6), (192, 136),
                                   (256, 256), (256, 2)])
def test_every_width(d, dim, interleaved, dtype):
  rot = rotary.make_rotary(dim, interleaved=interleaved, device=DEV)
  freq, _ = rotary.frequencies(dim)
  positions = torch.tensor([[0, 1, 2, 500, 7], [100000, 3, -4, 1, 999]], device=DEV)
  q, k = _rows(2, 5, 5, d, dtype, 0, False), _rows(2, 2, 5, d, dtype, 1)
  out_q, out_k = rotary.rotate(rot, positions, q, k)
  _check(out_q, q, positions, freq, interleaved=interleaved)
  _check(out_k, k, positions, freq, interleaved=interleaved)
  assert out_q.stride() == q.stride() and out_k.stride() == k.stride()  # results lie as the inputs do
  assert torch.equal(out_q[..., dim:], q[..., dim:])


@pytest.mark.parametrize("heads", [1, 3, 4, 5, 33])
@pytest.mark.parametrize("t", [1, 2, 63, 257])
def test_heads_and_tokens_of_every_number(heads, t):
  rot = rotary.make_rotary(64, device=DEV)
  freq, _ = rotary.frequencies(64)
  positions = torch.arange(t, device=DEV)[None] + torch.tensor([[5], [0], [1234]], device=DEV)
  q = _rows(3, heads, t, 64, torch.bfloat16, t)
  _check(rotary.rotate(rot, positions, q), q, positions, freq)


@pytest.mark.parametrize("scaling", [None, rotary.Scaling("linear", factor=4.0), rotary.Scaling("base", factor=8.0),
                                     rotary.Scaling("by_parts", factor=16.0, original=4096),
                                     rotary.Scaling("by_parts", factor=16.0, original=4096, attention=0.5),
                                     rotary.Scaling("bands", factor=8.0, original=8192)])
def test_far_positions_and_scalings(scaling):
  """2^-21 of the pair at any position: the angle's error does not grow with it."""
  rot = rotary.make_rotary(128, base=500000.0, scaling=scaling, device=DEV)
  freq, factor = rotary.frequencies(128, base=500000.0, scaling=scaling)
  positions = torch.tensor([[0, 1, 131071, 10 ** 6, 2 ** 31 - 1, -(2 ** 31), 10 ** 9 + 7]], device=DEV)
  q = _rows(1, 2, 7, 128, torch.float32, 3)
  _check(rotary.rotate(rot, positions, q), q, positions, freq, factor=factor)
  _check(rotary.rotate(rot, positions.int(), q), q, positions, freq, factor=factor)


def test_sines_and_cosines_of_f32_rows_are_right_to_their_last_places():
  """Pairs (1, 0) become cosine and sine.  An angle is cut off at 2^-32 of a turn (pi 2^-31), what it is beyond whole quarters rounded to
  24 bits (2^-24 of it, and so at most of a sine that is near 0, or of one above 0.7), sine and cosine to 2 units in the last place
  (2^-22): below pi 2^-31 + 2^-21 of each."""
  freq = [math.pi / 2 * (n % 4) + 1e-4 * n * n for n in range(1, 33)]  # close to the axes, and farther from them as positions grow
  positions = torch.arange(-300, 300, device=DEV)
  q = torch.zeros(1, 1, 600, 64, device=DEV)
  q[..., :32] = 1.0
  out = rotary.rotate(rotary.make_rotary(64, frequency=freq, device=DEV), positions, q)[0, 0].cpu().double()
  angle = rotary_ref.angles(positions.cpu(), freq)
  for got, want in ((out[:, :32], angle.cos()), (out[:, 32:], angle.sin())):
    assert ((got - want).abs() <= math.pi * 2.0 ** -31 + 2.0 ** -21 * want.abs() + 1e-15).all()


def test_given_frequencies_whole_turns_and_the_factor():
  freq = np.array([0.0, math.pi / 2, 2 * math.pi, -1.0])  # none, a quarter, (almost) a whole one, backwards
  rot = rotary.make_rotary(8, frequency=torch.tensor(freq), factor=-2.0, device=DEV)
  positions = torch.arange(9, device=DEV)
  q = _rows(2, 2, 9, 8, torch.float32, 4)
  _check(rotary.rotate(rot, positions, q), q, positions[None].expand(2, -1), freq, factor=-2.0)


def test_positions_of_every_kind():
  rot = rotary.make_rotary(64, device=DEV)
  q = _rows(3, 2, 40, 64, torch.float16, 0)
  positions = torch.arange(40, device=DEV) * 3
  want = rotary.rotate(rot, positions[None].expand(3, -1).contiguous(), q)
  odd = torch.zeros(3, 81, dtype=torch.int32, device=DEV)[:, 1::2]
  odd.copy_(positions[None])
  for p in (positions, positions[None], positions.int(), positions[None].expand(3, -1), odd):
    assert torch.equal(rotary.rotate(rot, p, q), want)


def test_operands_through_their_strides():
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(30, device=DEV)
  qkv = torch.randn(2, 30, 9, 72, device=DEV, dtype=torch.bfloat16)
  q, k = qkv[:, :, 2:6, :64].transpose(1, 2), qkv[:, :, 6:8, :64].transpose(1, 2)
  want = rotary.rotate(rot, positions, q.contiguous(), k.contiguous())
  got = rotary.rotate(rot, positions, q, k)
  assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
  odd = torch.zeros(2, 4, 30, 67, device=DEV, dtype=torch.bfloat16)[..., 3:]  # rows that start between 16-byte boundaries
  odd.copy_(q)
  assert torch.equal(rotary.rotate(rot, positions, odd), want[0])
  wide = q[:1, :1].expand(2, 4, -1, -1)  # one head for all
  assert torch.equal(rotary.rotate(rot, positions, wide), want[0][:1, :1].expand(2, 4, -1, -1))
  flipped = q.transpose(2, 3).contiguous().transpose(2, 3)  # tokens contiguous
  assert torch.equal(rotary.rotate(rot, positions, flipped), want[0])


def test_results_of_parts_of_a_projection_lie_as_the_projection_does():
  rot = rotary.make_rotary(64, device=DEV)
  qkv = torch.randn(2, 30, 8, 64, device=DEV, dtype=torch.bfloat16)
  q, k = qkv[:, :, :6].transpose(1, 2), qkv[:, :, 6:].transpose(1, 2)
  out_q, out_k = rotary.rotate(rot, torch.arange(30, device=DEV), q, k)
  assert out_q.transpose(1, 2).is_contiguous() and out_k.transpose(1, 2).is_contiguous()
  assert out_q.stride() == torch.empty_like(q).stride()


def test_a_module_that_holds_one_is_copied_and_pickled():
  rot = rotary.make_rotary(32, base=500.0, interleaved=True, factor=1.5, device=DEV)
  q, positions = _rows(1, 2, 9, 48, torch.float32, 5), torch.arange(9, device=DEV) * 1000
  want = rotary.rotate(rot, positions, q)
  for other in (copy.deepcopy(rot), copy.copy(rot), pickle.loads(pickle.dumps(rot))):
    assert torch.equal(rotary.rotate(other, positions, q), want)
  assert copy.deepcopy(rot).turns.data_ptr() != rot.turns.data_ptr()


def test_rows_without_gradients_stay_so():
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(5, device=DEV)
  q, k = _rows(1, 2, 5, 64, torch.float32, 6).requires_grad_(), _rows(1, 1, 5, 64, torch.float32, 7)
  out_q, out_k = rotary.rotate(rot, positions, q, k)
  assert out_q.requires_grad and not out_k.requires_grad
  (out_q.sum() + out_k.sum()).backward()
  grad, q.grad = q.grad, None
  rotary.rotate(rot, positions, q).sum().backward()
  assert torch.equal(q.grad, grad)
  out_k, out_q = rotary.rotate(rot, positions, k, q)
  assert out_q.requires_grad and not out_k.requires_grad
  q.grad = None
  out_q.sum().backward()
  assert torch.equal(q.grad, grad) and k.grad is None


def test_nothing_at_all():
  rot = rotary.make_rotary(64, device=DEV)
  q, k = torch.zeros(2, 4, 0, 64, device=DEV), torch.zeros(2, 0, 0, 64, device=DEV)
  out = rotary.rotate(rot, torch.zeros(2, 0, dtype=torch.int64, device=DEV), q, k)
  assert out[0].shape == q.shape and out[1].shape == k.shape
  q = torch.randn(2, 4, 3, 64, device=DEV)
  out = rotary.rotate(rot, torch.arange(3, device=DEV), q, q[:, :0])
  assert torch.equal(out[0], rotary.rotate(rot, torch.arange(3, device=DEV), q)) and out[1].shape == (2, 0, 3, 64)
  assert rotary.rotate(rot, torch.arange(3, device=DEV), q[:0]).shape == (0, 4, 3, 64)


def test_channels_that_are_copied_are_copied_bit_for_bit():
  rot = rotary.make_rotary(32, device=DEV)
  q = torch.randint(0, 2 ** 16, (1, 2, 5, 64), device=DEV, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)  # NaN and infinities among them
  out = rotary.rotate(rot, torch.arange(5, device=DEV), q)
  assert torch.equal(out.view(torch.int16)[..., 32:], q.view(torch.int16)[..., 32:])


# ----------------------------------------------------------------------------------------------
# gradients
# ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved,d,dim", [(False, 128, 128), (True, 80, 40), (True, 64, 64), (False, 80, 20)])
def test_gradients_are_the_rotation_back(interleaved, d, dim, dtype):
  rot = rotary.make_rotary(dim, interleaved=interleaved, factor=1.5, device=DEV)
  freq, _ = rotary.frequencies(dim)
  positions = torch.tensor([[3, 70000, 11], [0, 1, 2]], device=DEV)
  q, k = _rows(2, 4, 3, d, dtype, 0).requires_grad_(True), _rows(2, 2, 3, d, dtype, 1, False).requires_grad_(True)
  out = rotary.rotate(rot, positions, q, k)
  dq, dk = _rows(2, 4, 3, d, dtype, 2, False), _rows(2, 2, 3, d, dtype, 3)
  torch.autograd.backward(out, (dq, dk))
  _check(q.grad, dq, positions, freq, interleaved=interleaved, factor=1.5, inverse=True)
  _check(k.grad, dk, positions, freq, interleaved=interleaved, factor=1.5, inverse=True)


def test_gradients_against_differences():
  """The rotation is linear: <rotate(x + h) - rotate(x), g> = <h, gradient>, but for roundings of 2^-21 of some 4000 terms of size 1."""
  rot = rotary.make_rotary(48, interleaved=True, factor=0.7, device=DEV)
  positions = torch.arange(17, device=DEV) * 1001
  x, h, g = (_rows(1, 4, 17, 64, torch.float32, i) for i in range(3))
  leaf = x.clone().requires_grad_(True)
  (rotary.rotate(rot, positions, leaf) * g).sum().backward()
  change = (rotary.rotate(rot, positions, x + h).double() - rotary.rotate(rot, positions, x).double()) * g.double()
  want = (h.double() * leaf.grad.double()).sum()
  assert abs(float(change.sum() - want)) <= 4352 * 4 * 2.0 ** -21 * 3


def test_gradients_of_one_side_only_and_of_gradients():
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(6, device=DEV)
  q, k = _rows(1, 2, 6, 64, torch.float32, 0), _rows(1, 1, 6, 64, torch.float32, 1)
  lq, lk = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
  both = rotary.rotate(rot, positions, lq, lk)
  (want_k,) = torch.autograd.grad(both[1].sum(), lk, retain_graph=True)  # q's output has no part
  out = rotary.rotate(rot, positions, q, lk)
  assert out[1].requires_grad
  out[1].sum().backward()
  assert torch.equal(lk.grad, want_k)
  assert torch.autograd.grad(both[1].sum(), lq, allow_unused=True, retain_graph=True)[0] is None
  # twice: the gradient of (y . y) / 2 is x again, and its gradient the identity's
  y = rotary.rotate(rot, positions, lq)
  (first,) = torch.autograd.grad((y * y).sum() / 2, lq, create_graph=True)
  assert (first - lq).abs().max() <= 2.0 ** -19 * q.abs().max()
  (second,) = torch.autograd.grad(first.sum(), lq)
  assert (second - 1).abs().max() <= 2.0 ** -18
  with torch.no_grad():
    assert not rotary.rotate(rot, positions, lq).requires_grad


def test_positions_that_change_before_the_backward_are_noticed():
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(6, device=DEV)
  q = _rows(1, 2, 6, 64, torch.float32, 0).requires_grad_(True)
  out = rotary.rotate(rot, positions, q)
  positions += 1
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    out.sum().backward()


def test_saved_positions_go_through_hooks():
  """What a hook gives back is read if it is positions still, on the device, and refused before a kernel follows its address if not."""
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(12, device=DEV).view(2, 6) * 100
  q, g = _rows(2, 2, 6, 64, torch.float32, 0).requires_grad_(True), _rows(2, 2, 6, 64, torch.float32, 1)

  def gradient(unpack):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
      out = rotary.rotate(rot, positions, q)
    return torch.autograd.grad(out, q, g)[0]

  want = gradient(lambda t: t.to(DEV))
  assert torch.equal(want, torch.autograd.grad(rotary.rotate(rot, positions, q), q, g)[0])
  assert torch.equal(want, gradient(lambda t: t.to(DEV).int()))
  assert torch.equal(want, gradient(lambda t: t.t().contiguous().to(DEV).t()))
  for unpack, message in ((lambda t: t, "positions are on cpu"), (lambda t: t.to(DEV).half(), "int32 or int64"), (lambda t: t.to(DEV)[:, :5], "do not match"),
                          (lambda t: t.to(DEV)[0, 0], "expected q and k")):
    with pytest.raises(ValueError, match=message):
      gradient(unpack)


def test_shared_heads_and_broadcast_inputs():
  """Gradients of a head that is expanded add up; a gradient that is expanded itself is read."""
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(6, device=DEV)
  one = _rows(2, 1, 6, 64, torch.float32, 0).requires_grad_(True)
  rotary.rotate(rot, positions, one.expand(-1, 4, -1, -1)).sum().backward()
  back, _ = rotary_ref.rotate(torch.ones(2, 1, 6, 64), positions[None].expand(2, -1), rotary.frequencies(64)[0], inverse=True)
  assert (one.grad.cpu().double() - 4 * back).abs().max() <= 8 * 2.0 ** -21


# ----------------------------------------------------------------------------------------------
# where it runs
# ----------------------------------------------------------------------------------------------
def test_streams_and_graphs():
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(12, device=DEV)
  q, k = _rows(2, 4, 12, 64, torch.bfloat16, 0), _rows(2, 2, 12, 64, torch.bfloat16, 1)
  want = rotary.rotate(rot, positions, q, k)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    got = rotary.rotate(rot, positions, q, k)
  torch.cuda.current_stream().wait_stream(side)
  assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = rotary.rotate(rot, positions, q, k)
  for step in (0, 5):
    positions += step
    graph.replay()
    want = rotary.rotate(rot, positions, q, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_captured_training_step():
  rot = rotary.make_rotary(64, device=DEV)
  positions = torch.arange(12, device=DEV)
  q, g = _rows(2, 4, 12, 64, torch.float32, 0), _rows(2, 4, 12, 64, torch.float32, 1)

  def step():
    leaf = q.detach().requires_grad_(True)
    return torch.autograd.grad(rotary.rotate(rot, positions, leaf), leaf, g)[0]

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = step()
  positions += 3
  g.mul_(2)
  graph.replay()
  assert torch.equal(got, step())


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_calls_give_the_same(backend):
  rot, positions = rotary.make_rotary(64, device=DEV), torch.arange(6, device=DEV)

  def step(q, k):
    out_q, out_k = rotary.rotate(rot, positions, q * 0.5, k)
    return out_q.sum(1) + 2.0 * out_k.sum(1)

  results = []
  for call in (step, torch.compile(step, backend=backend)):
    q, k = _rows(2, 4, 6, 64, torch.float32, 0).requires_grad_(True), _rows(2, 2, 6, 64, torch.float32, 1, False).requires_grad_(True)
    out = call(q, k)
    results.append((out, *torch.autograd.grad(out.square().sum(), (q, k))))
  assert all(torch.equal(a, b) for a, b in zip(*results))
  with torch.no_grad():
    assert torch.equal(torch.compile(step, backend=backend)(q, k), out)


def test_transforms_are_refused():
  rot, positions, q = rotary.make_rotary(64, device=DEV), torch.arange(6, device=DEV), _rows(2, 4, 6, 64, torch.float32, 0)
  call = lambda x: rotary.rotate(rot, positions, x)  # noqa: E731
  for transform in (lambda: torch.func.grad(lambda x: call(x).sum())(q), lambda: torch.func.vjp(call, q), lambda: torch.func.jvp(call, (q,), (q,)),
                    lambda: torch.func.vmap(call)(q[None]), lambda: torch.func.vmap(lambda p: rotary.rotate(rot, p, q))(positions[None])):
    with pytest.raises((RuntimeError, NotImplementedError)):
      transform()


def test_offsets_beyond_32_bits():
  """The last rows of a tensor of over 2^32 bytes."""
  rot = rotary.make_rotary(64, device=DEV)
  q = torch.empty(1, 1, (1 << 25) + 5, 64, dtype=torch.bfloat16, device=DEV)  # 4.3 GB
  q[:, :, -5:] = _rows(1, 1, 5, 64, torch.bfloat16, 0)
  q[:, :, :-5] = 0
  positions = torch.zeros(1, q.shape[2], dtype=torch.int32, device=DEV)
  positions[:, -5:] = torch.arange(5, device=DEV) + 100
  out = rotary.rotate(rot, positions, q)
  assert torch.equal(out[:, :, -5:], rotary.rotate(rot, positions[:, -5:], q[:, :, -5:].contiguous())) and not out[:, :, :-5].any()


@pytest.mark.parametrize("grad", [False, True])
def test_rows_without_memory_are_refused(grad):
  """They have an address of nothing; a call would give back memory that nobody wrote."""
  rot, positions = rotary.make_rotary(64, device=DEV), torch.arange(3, device=DEV)
  q = torch.randn(2, 4, 3, 64, device=DEV).requires_grad_(grad)
  with pytest.raises((ValueError, RuntimeError)):
    torch.func.functionalize(lambda x: rotary.rotate(rot, positions, x))(q)
  with FakeTensorMode(allow_non_fake_inputs=True) as mode, pytest.raises((ValueError, RuntimeError)):
    rotary.rotate(rot, positions, mode.from_tensor(q))
  with FakeTensorMode(allow_non_fake_inputs=True) as mode, pytest.raises((ValueError, RuntimeError)):
    rotary.rotate(rot, positions, q, mode.from_tensor(q))


def test_refusals():
  rot = rotary.make_rotary(64, device=DEV)
  q, positions = torch.zeros(2, 4, 3, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int64, device=DEV)
  with pytest.raises(ValueError, match="positions are on"):
    rotary.rotate(rot, positions.cpu(), q)
  with pytest.raises(ValueError, match="rotary table"):
    rotary.rotate(rotary.make_rotary(64, device="cpu"), positions, q)
  with pytest.raises(RuntimeError, match="CUDA"):
    rotary.rotate(rot, positions, q, q.cpu())
  with pytest.raises(NotImplementedError, match="256"):
    rotary.rotate(rot, positions, torch.zeros(2, 4, 3, 264, device=DEV, dtype=torch.bfloat16))
