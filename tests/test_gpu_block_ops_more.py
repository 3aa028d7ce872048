"""Layer norm, linear and several-axis rotary operators: float32 operands of any stride and alignment, calls from several threads
at once, tensors on a device that is not the current one."""
import threading

import pytest
import torch

from pom_b200.operators import apply_rope_axes, layer_norm, linear
from tests.test_gpu_block_ops import BF, F32, block_pass, block_tensors, linear_check, linear_inputs, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 9, 16, 40, 700])
@pytest.mark.parametrize("K, N", [(64, 40), (136, 200), (257, 33), (1160, 520)])
def test_float32_strides_and_alignment(K, N, M):
    """Rows of wider matrices at offsets that 16-byte access can and cannot take, for x, weight, bias, residual and dy; the
    products on the few-row kernel, on the FMA kernel (short or small) and on the tensor cores."""
    _, _, b, _, _ = linear_inputs(M, K, N, F32, seed=3)
    xs, ws, rs = rand(M, K + 12, seed=4), rand(N, K + 12, seed=5, scale=K ** -0.5), rand(M, N + 12, seed=6)
    dys, bs = rand(M, N + 12, seed=7), rand(N + 1, seed=8)
    for at in (0, 4, 1, 7):
        x, w, r, dy = xs[:, at:at + K], ws[:, at:at + K], rs[:, at:at + N], dys[:, at:at + N]
        linear_check(x, w, bs[1:], r, "silu", dy, label=f"{at} ")
        linear_check(x, ws[:, :K].contiguous(), b, None, None, dy, label=f"x {at} ")
        linear_check(xs[:, :K].contiguous(), w, None, r, "gelu", dys[:, :N].contiguous(), label=f"w {at} ")
    x, w = rand(K, M, seed=9).t(), rand(K, N, seed=10, scale=K ** -0.5).t()  # columns side by side: copied
    linear_check(x, w, b, rs[:, :N].t().contiguous().t(), "gelu_tanh", dys[:, :N].t().contiguous().t(), label="columns ")


def test_threads_that_check_positions_at_once():
    """Each thread on its own stream, with its own positions: every answer is the thread's own, from its first call on."""
    tables = [(torch.ones(10, 4, device="cuda"), torch.zeros(10, 4, device="cuda"))]
    x = rand(1, 64, 16, dtype=BF)
    torch.cuda.synchronize()
    ready, wrong = threading.Barrier(6), []

    def work(i):
        pos = torch.full((64, 1), i, device="cuda")
        bad = torch.full((64, 1), 10 + i, device="cuda")
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.synchronize()
            ready.wait()
            for _ in range(50):
                try:
                    if not torch.equal(apply_rope_axes(x, pos, tables), x):
                        wrong.append((i, "value"))
                    try:
                        apply_rope_axes(x, bad, tables)
                        wrong.append((i, "not refused"))
                    except IndexError as e:
                        if f"[{10 + i}, {10 + i}]" not in str(e):
                            wrong.append((i, str(e)))
                except Exception as e:  # noqa: BLE001
                    wrong.append((i, repr(e)))
            torch.cuda.current_stream().synchronize()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not wrong, wrong[:5]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_threads_that_run_a_block_at_once(dtype):
    sets = [block_tensors(dtype, seed=100 * i) for i in range(3)]
    want = [block_pass(t) for t in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = block_pass(sets[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not wrong


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
@pytest.mark.parametrize("dtype", [BF, F32])
def test_block_on_the_device_that_is_not_current(dtype):
    torch.cuda.set_device(0)
    t = block_tensors(dtype)
    want = [a.cpu() for a in block_pass(t)]
    there = {k: [(c.to("cuda:1"), s.to("cuda:1")) for c, s in v] if k == "tables" else
             v.detach().to("cuda:1").requires_grad_(v.requires_grad) for k, v in t.items()}
    got = block_pass(there)
    assert torch.cuda.current_device() == 0
    for a, b in zip(got, want):
        assert a.device.index == 1 and torch.equal(a.cpu(), b)
    checked = apply_rope_axes(there["x"].detach(), there["pos"], there["tables"])
    assert torch.equal(checked, apply_rope_axes(there["x"].detach(), there["pos"], there["tables"], validate=False))
    with pytest.raises(RuntimeError, match="same GPU"):
        layer_norm(there["x"], t["nw"])
    with pytest.raises(RuntimeError, match="same GPU"):
        linear(there["x"], t["w1"])


def test_a_default_device_does_not_move_the_host_memory():
    """torch.set_default_device("cuda") must not decide where the range of the positions goes."""
    tables = [(torch.ones(10, 4, device="cuda"), torch.zeros(10, 4, device="cuda"))]
    x, pos = rand(1, 64, 16, dtype=BF), torch.full((64, 1), 7, device="cuda")
    got = []

    def work():  # a new thread: its memory is not made yet
        try:
            with torch.device("cuda"):
                got.append(apply_rope_axes(x, pos, tables))
        except Exception as e:  # noqa: BLE001
            got.append(repr(e))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert isinstance(got[0], torch.Tensor) and torch.equal(got[0], x), got


def test_positions_are_waited_for_on_a_stream_that_is_behind():
    """Longer than the call looks at the host's memory: it waits for its own stream, and another stream's work does not count."""
    tables = [(torch.ones(10, 4, device="cuda"), torch.zeros(10, 4, device="cuda"))]
    x, good, bad = rand(1, 64, 16, dtype=BF), torch.full((64, 1), 9, device="cuda"), torch.full((64, 1), 12, device="cuda")
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            torch.cuda._sleep(4_000_000)  # some 2 ms
            assert torch.equal(apply_rope_axes(x, good, tables), x)
            torch.cuda._sleep(4_000_000)
            with pytest.raises(IndexError, match=r"\[12, 12\]"):
                apply_rope_axes(x, bad, tables)
