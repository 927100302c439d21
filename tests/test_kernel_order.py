"""Kernels start beside the last blocks of the kernel ahead and may read what it writes only behind their wait for it.

Without a device: no kernel takes anything but weights, tables and pure outputs through ``__restrict__`` parameters (the compiler takes it that what a const one points to
never changes while the kernel runs, and may move its loads ahead of the wait) or reads by ``__ldg``.  On the device: every kind of kernel right behind a product of some 20 us that writes its input, launched one by one and
replayed from a graph, against the same numbers when nothing runs any more."""
import re
from pathlib import Path

import pytest
import torch

from spyinfer_b200 import kernels

DEV = "cuda:0"
gpu = pytest.mark.gpu

# parameters that are weights or tables of the model
WEIGHTS = {"table", "pairs", "w", "weight", "y_weight", "q_w", "k_w", "q_weight", "k_weight", "wq", "wc", "rope", "cos_sin", "inv_freq", "bias", "z_bias", "x_bias", "dt_bias",
           "a_log", "d_skip", "kernel", "a_weight", "b_weight", "a_w", "a_bias", "temp", "W", "next_weights", "row"}
# parameters that a kernel only writes (the table: by the kernel that makes it; the workspace: what its own blocks hand one another, by loads that pass the first cache)
OUTPUTS = {"out", "pages", "pooled", "q_out", "pieces", "workspace", "y", "weights_out", "choice", "choice_w", "shared_w", "counts", "offsets", "slot", "row_token", "row_w",
           "tile_expert", "codes", "scales", "copy", "floor_out", "slice_v", "slice_i", "tokens", "C", "cq_out", "table"}


def code_of(path):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def test_only_weights_and_outputs_are_restrict_parameters():
    folder = Path(kernels.__file__).parent / "csrc"
    seen = 0
    for path in sorted(folder.glob("*.cu")) + sorted(folder.glob("*.cuh")):
        for const, name in re.findall(r"(const )?[A-Za-z_][A-Za-z0-9_]*\s*\*\s*__restrict__\s+([A-Za-z0-9_]+)(?=\s*[,)])", code_of(path)):
            seen += 1
            assert name in (WEIGHTS if const else OUTPUTS), f"{path.name}: {const}... * __restrict__ {name}"
    assert seen > 100


def test_no_read_only_loads_of_data():
    folder = Path(kernels.__file__).parent / "csrc"
    for path in sorted(folder.glob("*.cu")) + sorted(folder.glob("*.cuh")):
        for what in re.findall(r"__ldg\(([^;]*?)\)|ld\.global\.nc", code_of(path)):
            assert what.startswith(("p.scores.sinks", "p.scores.slopes")), f"{path.name}: {what}"      # the heads' weights


def right_behind(consume, dtype=torch.bfloat16, before=lambda: None, M=64, N=24576, K=4096):
    """``consume(z)`` of what the product ``z [M, N]`` writes; ``before`` runs ahead of the product."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(M, K, generator=g, device=DEV).to(torch.bfloat16)
    w = (torch.randn(N, K, generator=g, device=DEV) / K ** 0.5).to(torch.bfloat16)
    z = torch.empty(M, N, dtype=dtype, device=DEV)

    def run():
        before()
        kernels.gemm_tcgen05(x, w, out=z)
        return consume(z)

    def flat(out):
        return out if isinstance(out, (tuple, list)) else (out,)

    run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = run()
        for i in range(6):
            x.copy_(torch.randn(M, K, generator=g, device=DEV))
            z.zero_()
            if i % 2:
                graph.replay()
                got = held
            else:
                got = run()
            side.synchronize()
            got = [t.clone() for t in flat(got)]
            kept = z.clone()
            side.synchronize()
            before()
            side.synchronize()
            want = flat(consume(kept))
            side.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b), f"pass {i}: {int((a != b).sum())} of {a.numel()} differ"


def rows_of(z, rows, length):
    return z.view(-1)[:rows * length].view(rows, length)


def new(rows, length, dtype=torch.bfloat16):
    return torch.empty(rows, length, dtype=dtype, device=DEV)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,length", [(64, 4096), (384, 4096), (1500, 1024), (300, 4999), (1, 5120)])
def test_norms_right_behind_a_product(rows, length, dtype):
    weight = (1 + 0.1 * torch.randn(length, device=DEV)).to(torch.bfloat16)
    stream = torch.randn(rows, length, device=DEV)
    right_behind(lambda z: kernels.rmsnorm(stream, weight, 1e-6, new(rows, length), delta=rows_of(z, rows, length)), dtype)
    right_behind(lambda z: kernels.rmsnorm(rows_of(z, rows, length), weight, 1e-6, new(rows, length)), dtype)
    right_behind(lambda z: kernels.layernorm(stream, weight, 1e-6, new(rows, length), delta=rows_of(z, rows, length)), dtype)

    h, copy = stream.clone(), new(rows, length)

    def added(z):
        kernels.residual_norm(h, rows_of(z, rows, length), weight, 1e-6, copy=copy)
        return h, copy

    def summed(z):
        return kernels.stream_sum(h, rows_of(z, rows, length), copy=copy), copy

    def grouped(z):
        kernels.group_norm(h, 1, 1e-6, y=rows_of(z, rows, length), y_weight=weight, weight=weight, out=copy)
        return h, copy

    for consume in (added, summed, grouped):
        right_behind(consume, dtype, before=lambda: h.copy_(stream))
    right_behind(lambda z: kernels.scaled_sum(new(rows, length, torch.float32), rows_of(z, rows, length), 0.5, rows_of(z, rows, length), 2.0), dtype)
    w32 = weight.float()
    right_behind(lambda z: kernels.normed_sum(new(rows, length, torch.float32), rows_of(z, rows, length), w32, 0.5, rows_of(z, rows, length), w32, 2.0, 1e-6), dtype)
    if dtype == torch.float32:
        half = rows // 2 or 1
        right_behind(lambda z: kernels.rmsnorm(stream[:half], weight, 1e-6, new(half, length), delta=z.view(-1)[:2 * half * length].view(2, half, length)), dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,length", [(64, 12288), (384, 2048), (300, 2499), (1, 4096)])
def test_activations_right_behind_a_product(rows, length, dtype):
    def two(z):
        return rows_of(z, rows, 2 * length)

    right_behind(lambda z: kernels.swiglu(two(z), new(rows, length, dtype)), dtype)
    right_behind(lambda z: kernels.gated_activation(two(z), new(rows, length, dtype), "gelu_tanh"), dtype)
    right_behind(lambda z: kernels.activation(rows_of(z, rows, length), new(rows, length, dtype), "relu2"), dtype)
    right_behind(lambda z: kernels.clamped_glu(two(z), None, new(rows, length, torch.bfloat16), 7.0, 1.702), dtype)


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (40, 1000, 1024), (300, 512, 4096), (5, 40, 24576)])
def test_products_right_behind_a_product(M, N, K):
    w32 = torch.randn(N, K, device=DEV) / K ** 0.5
    w16 = w32.to(torch.bfloat16)
    right_behind(lambda z: kernels.gemm_simt(rows_of(z, M, K), w32, new(M, N, torch.float32)), torch.float32)
    right_behind(lambda z: kernels.gemm_simt(rows_of(z, M, K), w16, new(M, N, torch.float32)), torch.float32)
    right_behind(lambda z: kernels.gemm_simt(rows_of(z, M, K), w16, new(M, N)), torch.bfloat16)
    if kernels.gemm_split_takes(w16):
        right_behind(lambda z: kernels.gemm_split(rows_of(z, M, K), w16, new(M, N, torch.float32)), torch.float32)
    right_behind(lambda z: kernels.gemm_tcgen05(rows_of(z, M, K), w16, out_dtype=torch.float32), torch.bfloat16)


@gpu
def test_what_follows_a_recurrence_right_behind_a_product():
    rows, size = 96, 4096
    proj, o, weight = torch.randn(rows, size, device=DEV), torch.randn(rows, size, device=DEV), torch.ones(size, device=DEV)
    for pair in (lambda z: (rows_of(z, rows, size), proj), lambda z: (o, rows_of(z, rows, size))):
        right_behind(lambda z: kernels.gated_head_norm(*pair(z), 0, weight, new(rows, size), 32, 128, 1e-6, "silu"), torch.float32)
        right_behind(lambda z: kernels.gate_group_norm(*pair(z), 0, weight, new(rows, size), 8, 1e-6), torch.float32)
    right_behind(lambda z: kernels.tanh_cols(rows_of(z, rows, size), 128, 512, new(rows, 512)), torch.float32)


@gpu
@pytest.mark.parametrize("tokens,experts,top", [(64, 64, 4), (1000, 128, 8), (7, 16, 2)])
def test_router_and_gather_right_behind_a_product(tokens, experts, top):
    x = torch.randn(tokens, 256, device=DEV).to(torch.bfloat16)

    def routed(z):
        offsets, slot, row_token, row_w, shared_w = kernels.moe_route(rows_of(z, tokens, experts + 1), experts, top, True)
        return offsets, slot, row_token, row_w, shared_w, kernels.gather_rows(x, row_token, new(tokens * top, 256))

    right_behind(routed, torch.float32)


@gpu
def test_sampling_and_its_tokens_embedding_right_behind_a_product():
    """The logits' largest, and the rows of the tokens that the kernel ahead has chosen; and draws with temperatures and a top k."""
    table = torch.randn(24576, 512, device=DEV).to(torch.bfloat16)
    temperature, seed = torch.full((64,), 0.7, device=DEV), torch.arange(64, device=DEV)
    draw, top_k = torch.zeros(64, dtype=torch.int64, device=DEV), torch.full((64,), 20, dtype=torch.int32, device=DEV)

    def largest(z):
        tokens = kernels.sample(z, torch.empty(64, dtype=torch.int32, device=DEV))
        return tokens, kernels.embedding(table, tokens, new(64, 512, torch.float32))

    def drawn(z):
        tokens = kernels.sample(z, torch.empty(64, dtype=torch.int32, device=DEV), temperature, seed, draw, top_k)
        return tokens, kernels.embedding(table, tokens, new(64, 512, torch.float32))

    right_behind(largest, torch.float32)
    right_behind(drawn, torch.float32)
