"""Calls of the block's operators that their documentation allows besides the plain ones: from threads at
once, inside torch.compile, and a block's training step captured and replayed."""
import threading

import pytest
import torch

from dsalt.kernels import branch_norm, counter_dropout, gated_ffn
from dsalt.modules import DSALTTransformerBlock

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def operands(seed, rows):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s, std=1.0: (torch.randn(*s, device=DEV, generator=g) * std).to(BF)
    return {"x": rnd(rows, 72), "h": rnd(rows, 72), "w": rnd(72), "post": rnd(72), "gate": rnd(rows, 1),
            "wg": rnd(136, 72, std=0.1), "wu": rnd(136, 72, std=0.1), "wd": rnd(72, 136, std=0.1)}


def chain(t, seed):
    """The three operators as a block chains them."""
    x, h = branch_norm(t["x"], t["h"], t["w"], post_weight=t["post"], gate=t["gate"], residual_scale=0.9)
    f = gated_ffn(h, t["wg"], t["wu"], t["wd"])
    x, h = branch_norm(x, f, t["w"], p=0.2, seed=seed, offset=1)
    return x, counter_dropout(h, 0.1, seed, 2)


def step(t, seed):
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}
    outs = chain(leaves, seed)
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(leaves.values()), [torch.ones_like(o) for o in outs]))


def test_threads_with_streams_of_their_own():
    """Four threads, each on its own stream with its own operands, get what one thread gets."""
    cases = [(operands(i, rows), 100 + i) for i, rows in enumerate((3, 40, 300, 575))]
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = step(*cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # a thread's failure is the test's
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_inside_compile():
    t = operands(1, 50)
    want = step(t, 7)
    compiled = torch.compile(chain, backend="eager")
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}
    outs = compiled(leaves, 7)
    got = [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(leaves.values()), [torch.ones_like(o) for o in outs]))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("autocast", [False, True])
def test_block_training_step_in_a_graph(autocast):
    """A block with every option: forward and backward captured, replayed over new inputs and seeds with
    eager steps between, against eager results."""
    torch.manual_seed(3)
    b = DSALTTransformerBlock(128, 2, 4, 40, 4, 256, 264, layer_idx=1, post_norm=True, layer_scale=0.2, residual_scale=0.9,
                              fused_ffn=True, counter_dropout=True, dropout=0.1).to(DEV, FP if autocast else BF).train()
    twin = DSALTTransformerBlock(128, 2, 4, 40, 4, 256, 264, layer_idx=1, post_norm=True, layer_scale=0.2, residual_scale=0.9,
                                 fused_ffn=True, counter_dropout=True, dropout=0.1).to(DEV, FP if autocast else BF).train()
    twin.load_state_dict(b.state_dict())
    cu = torch.tensor([0, 200, 257, 388], dtype=torch.int32, device=DEV)
    x, seed = torch.randn(388, 128, device=DEV).to(BF), torch.tensor([1], device=DEV)

    def train(m, x, seed):
        xi = x.detach().requires_grad_()
        with torch.autocast("cuda", dtype=BF, enabled=autocast, cache_enabled=False):
            y, _, _ = m.join_branches(xi, m.attn_norm(xi), None, seed, cu_seqlens=cu, max_seqlen=256)
        ps = [xi, *m.parameters()]
        return y.detach(), *torch.autograd.grad(y, ps, torch.ones_like(y), allow_unused=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(twin, x, seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # twin's eager step holds no graph any more
        outs = train(twin, x, seed)
    for i in range(4):
        print(f"block replay {i} autocast={autocast}", flush=True)
        x.copy_(torch.randn(388, 128, device=DEV))
        seed.fill_(50 + i)
        graph.replay()
        want = train(b, x.clone(), 50 + i)
        assert len(outs) == len(want)
        for k, (p, q) in enumerate(zip(outs, want)):
            assert (p is None) == (q is None) and (p is None or torch.equal(p, q)), (i, k)
