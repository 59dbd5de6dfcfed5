"""The operators of a conditioned block where one call is not like the next:
tensors of more than 2^31 elements, calls queued one behind the other, and a
process whose first call is captured into a graph. A result is compared, bit by
bit, with that of the same rows alone, whose values the operators' own tests
hold to 64 bits."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_rotary_tokens_beyond_32_bits(cuda_device):
    from xgen_b200.ops import rope_axes

    s, h, d = 360001, 48, 128  # 2.2e9 channels
    q = torch.empty(1, s, h, d, device=cuda_device, dtype=torch.bfloat16).normal_()
    positions = torch.randint(0, 500, (s, 3), device=cuda_device)
    out, _ = rope_axes(q, None, positions, axes=(32, 48, 48))
    for rows in (slice(0, 9), slice(349520, 349531), slice(s - 7, s)):  # the second ends and begins behind 2^31
        alone, _ = rope_axes(q[:, rows], None, positions[rows], axes=(32, 48, 48))
        assert torch.equal(out[:, rows], alone)


@pytest.mark.parametrize("quant", [None, "int8"])
def test_norm_rows_beyond_32_bits(cuda_device, quant):
    from xgen_b200.ops import sandwich_norm

    s, w = 140001, 16384  # 2.3e9 channels
    y, x = (torch.empty(1, s, w, device=cuda_device, dtype=torch.bfloat16).normal_() for _ in range(2))
    got = sandwich_norm(y, x, pre_norm="layernorm", quant=quant)
    for rows in (slice(0, 400), slice(130900, 131300), slice(s - 400, s)):
        alone = sandwich_norm(y[:, rows], x[:, rows], pre_norm="layernorm", quant=quant)
        assert all(torch.equal(a[:, rows], b) for a, b in zip(got, alone))


def test_int8_rows_beyond_32_bits(cuda_device):
    from xgen_b200.int8_linear import int8_linear

    m, n, k = 140001, 16384, 256  # 2.3e9 results; the input is a view of wider rows
    wide = torch.empty(m, 16384, device=cuda_device, dtype=torch.bfloat16)
    x = wide[:, 512:512 + k].normal_()
    weight = torch.randint(-127, 128, (n, k), device=cuda_device, dtype=torch.int8)
    scale = 1e-3 * (1 + torch.rand(n, device=cuda_device))
    residual, gate = torch.empty(m, n, device=cuda_device, dtype=torch.bfloat16).normal_(), torch.randn(3, n, device=cuda_device).bfloat16()
    at = torch.randint(0, 3, (m,), device=cuda_device)
    got = int8_linear(x, weight, scale, gate=gate, gate_index=at, residual=residual)
    for rows in (slice(0, 300), slice(130900, 131300), slice(m - 300, m)):
        assert torch.equal(got[rows], int8_linear(x[rows], weight, scale, gate=gate, gate_index=at[rows], residual=residual[rows]))


@pytest.mark.parametrize("m", [3, 20, 200, 1000])
def test_int8_calls_one_behind_the_other(cuda_device, m):
    """The quantiser of a call, its product and the next call's quantiser (whose
    workspace is the first's) overlap at most as far as their data allow."""
    from xgen_b200.int8_linear import int8_linear

    g = torch.Generator(device=cuda_device).manual_seed(m)
    n, k = 1536, 5120
    weight = torch.randint(-127, 128, (n, k), generator=g, device=cuda_device, dtype=torch.int8)
    scale = 1e-3 * torch.rand(n, generator=g, device=cuda_device)
    xs = [torch.randn(m, k, generator=g, device=cuda_device).bfloat16() for _ in range(8)]
    alone = []
    for x in xs:
        torch.cuda.synchronize(cuda_device)
        alone.append(int8_linear(x, weight, scale))
    torch.cuda.synchronize(cuda_device)
    queued = [int8_linear(xs[i % 8], weight, scale) for i in range(120)]
    chained = xs[0]
    for _ in range(3):  # the input of a call is the last one's result
        chained = int8_linear(torch.cat([int8_linear(chained, weight, scale)] * 4, -1)[:, :k].contiguous(), weight, scale).repeat(1, 4)[:, :k]
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    torch.cuda.synchronize(cuda_device)
    both = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            both.append(int8_linear(xs[i % 8], weight, scale))
    torch.cuda.synchronize(cuda_device)
    for i, y in enumerate(queued):
        assert torch.equal(y, alone[i % 8]), i
    for i, y in enumerate(both):
        assert torch.equal(y, alone[i % 8]), i
    again = xs[0]
    for _ in range(3):
        torch.cuda.synchronize(cuda_device)
        inner = int8_linear(again, weight, scale)
        torch.cuda.synchronize(cuda_device)
        wide = torch.cat([inner] * 4, -1)[:, :k].contiguous()
        torch.cuda.synchronize(cuda_device)
        again = int8_linear(wide, weight, scale).repeat(1, 4)[:, :k]
    assert torch.equal(chained, again)


FIRST_CALL_CAPTURED = """
import torch
from xgen_b200.attention import cross_attention, kernel_errors
from xgen_b200.int8_linear import int8_linear
from xgen_b200.ops import rope_axes, sandwich_norm

dev = torch.device("cuda")
q, kv = torch.randn(2, 300, 4, 64, device=dev).half(), torch.randn(2, 77, 4, 64, device=dev).half()
x, w = torch.randn(600, 256, device=dev).half(), torch.randint(-127, 128, (256, 256), device=dev, dtype=torch.int8)
ws, at = torch.rand(256, device=dev), torch.randint(0, 90, (300, 2), device=dev)
mask = torch.rand(2, 77, device=dev) < 0.5

def run():
    t, _ = rope_axes(q, None, at, axes=(32, 32))
    a = cross_attention(t.transpose(1, 2), kv.transpose(1, 2), kv.transpose(1, 2), key_mask=mask)
    one = cross_attention(t[:, :1].transpose(1, 2), kv.transpose(1, 2), kv.transpose(1, 2), key_mask=mask)
    y = int8_linear(x, w, ws)
    few = int8_linear(x[:9], w, ws)
    return (t, a, one, y, few, *sandwich_norm(y[None], x[None], quant="int8"))

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
assert kernel_errors(dev) == 0
print("equal")
"""


def test_first_call_of_a_process_is_captured(cuda_device):
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=Path(__file__).resolve().parents[1], capture_output=True,
                         text=True, timeout=240)
    assert run.returncode == 0 and "equal" in run.stdout, run.stdout + run.stderr


ERROR_WORD_OF_A_CAPTURED_CALL = """
import torch
from xgen_b200 import attention, int8_linear

dev = torch.device("cuda")
seen, real = [], attention._err_ptr

def spy(index):
    seen.append(real(index))
    return seen[-1]

attention._err_ptr = int8_linear._err_ptr = spy
q, kv = torch.randn(1, 4, 300, 128, device=dev).bfloat16(), torch.randn(1, 4, 300, 128, device=dev).bfloat16()
x, w, ws = torch.randn(600, 256, device=dev).half(), torch.ones(256, 256, device=dev, dtype=torch.int8), torch.rand(256, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = [attention.dense_attention(q, kv, kv), attention.cross_attention(q, kv, kv), int8_linear.int8_linear(x, w, ws)]
word = attention._err_flag(dev)
assert len(seen) == 2 and seen[0] and set(seen) == {word.data_ptr()}, seen
assert attention.kernel_errors(dev) == 0  # nothing has run
word.fill_(5)  # what a wait that ran out would leave
graph.replay()
assert attention.kernel_errors(dev) == 5  # a replay does not clear it
word.zero_()
del graph, outs
torch.cuda.empty_cache()
again = [attention.cross_attention(q, kv, kv), int8_linear.int8_linear(x, w, ws)]
assert set(seen) == {word.data_ptr()} and attention.kernel_errors(dev) == 0
print("word")
"""


def test_a_first_captured_call_has_the_error_word(cuda_device):
    """A wait that gives up in a replayed graph is recorded where kernel_errors
    looks, also when the capture was the process's first call."""
    run = subprocess.run([sys.executable, "-c", ERROR_WORD_OF_A_CAPTURED_CALL], cwd=Path(__file__).resolve().parents[1], capture_output=True,
                         text=True, timeout=240)
    assert run.returncode == 0 and "word" in run.stdout, run.stdout + run.stderr
