"""The routed experts as a whole against their definition in 64 bits.

Where the tolerance comes from: a sum of n products in FP32 over the tensor cores' steps of 16 and the
warps is off by at most (n / 16 + 24) 2^-23 of the sum of its terms' sizes; an activation
keeps two BF16 terms (2^-16 of it are lost) and the output is rounded to BF16 (2^-8).  phi has slopes below 1.13.
"""

import math

import pytest
import torch

import cfm_b200  # noqa: F401
from cfm_b200.reader.progressive import channel_major_down
from cfm_b200.runtime.experts import PhaseContext, ProgressiveExperts, dense_routed_experts
from cfm_b200.runtime.fidelity import compare_logits, token_logprobs
from cfm_b200.runtime.routed import RoutedExperts, RoutedWorkspace
from cfm_b200.runtime.routing import route_tokens

pytestmark = pytest.mark.gpu


def layer(hidden, width, experts, seed=0, sigma=0.05):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    gate_up = torch.empty((experts, 2 * width, hidden), device="cuda", dtype=torch.bfloat16)
    down = torch.empty((experts, width, hidden), device="cuda", dtype=torch.bfloat16)
    gate_up.normal_(0.0, sigma, generator=generator)
    down.normal_(0.0, sigma, generator=generator)
    return gate_up, down.transpose(1, 2)


def batch(tokens, hidden, experts, top_k, seed=1, skew=0.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, hidden), device="cuda", generator=generator)
    x[:, ::97] *= 12.0
    logits = torch.randn((tokens, experts), device="cuda", generator=generator)
    logits += skew * torch.randn(experts, device="cuda", generator=generator)
    weights, ids = torch.softmax(logits, -1).topk(top_k, -1)
    return x.bfloat16(), ids.int().contiguous(), weights.contiguous()


def definition(gate_up, down, x, ids, weights, padding, activation):
    """The output in 64 bits and how far the kernels may be from it."""
    width, experts = down.shape[2], down.shape[0]
    x = x.double()
    out, allowed = torch.zeros_like(x), torch.zeros_like(x)
    up_step = (x.shape[1] / 16 + 24) * 2.0**-23
    down_step = (width / 8 + 24) * 2.0**-23
    for token in range(x.shape[0]):
        if padding is not None and padding[token]:
            continue
        for expert, weight in zip(ids[token].tolist(), weights[token].double()):
            if not 0 <= expert < experts:
                continue
            w, d = gate_up[expert].double(), down[expert].double()
            gate, up = (w @ x[token]).split(width)
            gate_off, up_off = (up_step * (w.abs() @ x[token].abs())).split(width)
            if activation == "silu":
                phi = gate * torch.sigmoid(gate)
            else:
                phi = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate**3)))
            a = phi * up
            off = 2.0**-16 * a.abs() + 1.13 * gate_off * up.abs() + (phi.abs() + 1.13 * gate_off) * up_off
            off = off + 2.0**-20 * a.abs() + 1e-30  # the exponential and the division
            out[token] += weight * (d @ a)
            allowed[token] += weight.abs() * (d.abs() @ (off + down_step * a.abs()))
    return out, allowed + 2.0**-8 * (out.abs() + allowed) + 1e-30


def check(gate_up, down, x, ids, weights, padding=None, activation="silu", run=None):
    run = run or RoutedExperts(gate_up, down, ids.shape[1], x.shape[0], activation=activation)
    got = run(x, ids, weights, padding)
    want, allowed = definition(gate_up, down, x, ids, weights, padding, activation)
    off = (got.double() - want).abs()
    run.check_status()
    assert got.dtype == torch.bfloat16 and (off <= allowed).all(), (off / allowed).max().item()
    return got


@pytest.mark.parametrize("tokens,hidden,width,experts,top_k", [
    (1, 128, 16, 1, 1), (1, 2048, 768, 16, 8), (2, 256, 48, 4, 4), (3, 384, 112, 7, 2),
    (8, 1152, 704, 8, 6), (9, 512, 32, 64, 4), (19, 1152, 176, 12, 6), (33, 640, 528, 5, 3),
    (40, 2176, 32, 4, 4), (70, 256, 64, 2, 1), (130, 384, 80, 3, 2), (2, 5120, 32, 4, 2),
    (20, 8320, 16, 2, 1), (34, 512, 208, 2, 1), (700, 256, 144, 5, 2), (260, 1024, 64, 1, 1), (3, 128, 4096, 2, 2), (300, 256, 16, 40, 8), (12, 256, 16, 300, 32),
])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_definition(tokens, hidden, width, experts, top_k, activation):
    gate_up, down = layer(hidden, width, experts)
    x, ids, weights = batch(tokens, hidden, experts, top_k)
    check(gate_up, down, x, ids, weights, activation=activation)


@pytest.mark.parametrize("tokens", [1, 5, 24, 90])
def test_types_padding_and_ids_without_an_expert(tokens):
    gate_up, down = layer(256, 96, 6)
    x, ids, weights = batch(tokens, 256, 6, 4, skew=2.0)
    ids[::3, 1] = -1
    ids[::4, 2] = 6
    ids[0] = 2**31 - 1
    padding = torch.arange(tokens, device="cuda") % 5 == 4
    x[padding] = math.nan  # padding rows are not read
    got = check(gate_up, down, x, ids, weights, padding)
    assert not got[0].any() and not got[padding].any()
    check(gate_up, down, x, ids.long(), weights.bfloat16(), padding)
    wide = ids.long()
    wide[0, 0] = 2**32 + 1  # an id that 32 bits would take for another
    wide[0, 1:] = -2**40
    assert not check(gate_up, down, x, wide, weights, padding)[0].any()


def test_all_rows_padding_or_without_an_expert():
    gate_up, down = layer(128, 32, 4)
    x, ids, weights = batch(7, 128, 4, 2)
    run = RoutedExperts(gate_up, down, 2, 16)
    out = torch.full_like(x, 3.0)
    assert run(x, ids, weights, torch.ones(7, device="cuda", dtype=torch.bool), out) is out
    assert not out.any()
    assert not run(x, torch.full_like(ids, -1), weights).any()


@pytest.mark.parametrize("tokens", [1, 5, 10, 50])
def test_the_same_expert_twice_and_one_expert_for_all(tokens):
    gate_up, down = layer(256, 48, 3)
    x, ids, weights = batch(tokens, 256, 3, 3)
    run = RoutedExperts(gate_up, down, 3, tokens)
    got = check(gate_up, down, x, torch.ones_like(ids), weights, run=run)
    assert torch.equal(run(x, torch.ones_like(ids), weights), got)
    ids[:, 2] = ids[:, 0]
    check(gate_up, down, x, ids, weights, run=run)


@pytest.mark.parametrize("tokens,top_k", [(16, 1), (8, 2), (1, 16), (2, 8), (1, 9), (17, 1), (6, 3), (1, 32), (32, 1)])
def test_few_pairs_and_one_more(tokens, top_k):
    gate_up, down = layer(384, 80, 40)
    x, ids, weights = batch(tokens, 384, 40, top_k)
    check(gate_up, down, x, ids, weights)
    check(gate_up, down, x, ids % 3, weights)  # many pairs per expert, most tokens with an expert twice
    check(gate_up, down, x, ids % 9, weights)


def test_a_tokens_output_does_not_depend_on_the_batch():
    """Among calls of up to 16 pairs, and among larger ones."""
    gate_up, down = layer(1152, 96, 4)
    x, ids, weights = batch(300, 1152, 4, 2)
    run = RoutedExperts(gate_up, down, 2, 300)
    for whole, parts in ((slice(0, 8), (slice(0, 1), slice(2, 7))),
                         (slice(0, 300), (slice(3, 20), slice(20, 52), slice(52, 180)))):
        out = run(x[whole], ids[whole], weights[whole])
        for rows in parts:
            assert torch.equal(run(x[rows], ids[rows], weights[rows]), out[rows])
        assert torch.equal(run(x[whole], ids[whole], weights[whole]), out)


def test_infinities_and_nan_stay_with_their_token():
    gate_up, down = layer(256, 48, 3)
    x, ids, weights = batch(12, 256, 3, 2)
    run = RoutedExperts(gate_up, down, 2, 12)
    clean = run(x, ids, weights)
    x[3, 7], x[9, 0] = math.nan, math.inf
    got = run(x, ids, weights)
    others = [t for t in range(12) if t not in (3, 9)]
    assert torch.equal(got[others], clean[others])
    assert got[3].isnan().all() and not got[9].isfinite().any()


def test_rows_behind_the_last_one_are_left_alone():
    gate_up, down = layer(128, 16, 4)
    x, ids, weights = batch(5, 128, 4, 2)
    buffer = torch.full((8, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    RoutedExperts(gate_up, down, 2, 8)(x, ids, weights, out=buffer[:5])
    assert (buffer[5:] == 7.0).all() and not (buffer[:5] == 7.0).all()


def test_layers_share_a_workspace_captured_and_on_another_stream():
    workspace = RoutedWorkspace(256, 48, 4, 2, 32, "cuda")
    layers = [layer(256, 48, 4, seed) for seed in (1, 2, 3)]
    runs = [RoutedExperts(g, d, 2, 32, workspace=workspace) for g, d in layers]
    x, ids, weights = batch(20, 256, 4, 2)
    padding = torch.zeros(20, device="cuda", dtype=torch.bool)
    want = [check(g, d, x, ids, weights, run=run) for (g, d), run in zip(layers, runs)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [run(x, ids, weights, padding) for run in runs]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for run in runs:  # graphs that share the workspace, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, run(x, ids, weights, padding)))
    more, ids2, weights2 = batch(20, 256, 4, 2, seed=9)
    for source, target in ((more, x), (ids2, ids), (weights2, weights)):
        target.copy_(source)
    padding[7] = True
    for graph, _ in graphs:
        graph.replay()
    for run, (_, out) in zip(runs, graphs):
        assert torch.equal(out, run(x, ids, weights, padding)) and not out[7].any()


def test_stock_rows_of_the_engine_side_caller():
    """Rows outside the policy, chunk by chunk, where the torch form stands otherwise."""
    gate_up, down = layer(256, 64, 8)
    x, ids, weights = batch(37, 256, 8, 2)
    run = RoutedExperts(gate_up, down, 2, 16)

    class Reader:
        max_tokens = 64

        def __call__(self, rows, ids, weights, padding=None, out=None, *, input_prepared=False):
            return rows * 0

    caller = ProgressiveExperts(Reader(), run.rows)
    out = caller.forward_modular(x, weights, ids, PhaseContext(num_decode_tokens=5))
    assert not out[:5].any()
    for rows in (slice(5, 21), slice(21, 37)):
        assert torch.equal(out[rows], run(x[rows], ids[rows], weights[rows]))
    # The torch form rounds gate and up to BF16 before the activation, and each expert's sum: 2^-8 of each.
    stock = dense_routed_experts(gate_up, down)(x, weights, ids)
    assert (out[5:].float() - stock[5:].float()).norm() < 0.02 * stock[5:].float().norm()
    assert run.rows(x[:0], weights[:0], ids[:0]).shape == (0, 256)


def test_weights_beyond_32_bits_of_elements():
    """The last expert of a layer whose gate and up rows are more than 2^31 elements."""
    hidden, width, experts = 8192, 1024, 130
    gate_up = torch.zeros((experts, 2 * width, hidden), device="cuda", dtype=torch.bfloat16)
    down = torch.zeros((experts, width, hidden), device="cuda", dtype=torch.bfloat16)
    assert gate_up[:-1].numel() > 2**31
    for expert in (0, experts - 1):
        for weight in (gate_up, down):
            weight[expert].normal_(0.0, 0.02, generator=torch.Generator(device="cuda").manual_seed(expert))
    small_gate_up, small_down = gate_up[[0, -1]], down[[0, -1]].transpose(1, 2)
    for tokens in (2, 20):
        x, ids, weights = batch(tokens, hidden, 2, 2)
        want = RoutedExperts(small_gate_up, small_down, 2, tokens)(x, ids, weights)
        got = RoutedExperts(gate_up, down.transpose(1, 2), 2, tokens)(x, ids * (experts - 1), weights)
        assert torch.equal(got, want) and got.any()


@pytest.mark.parametrize("tokens,experts,top_k", [(1024, 12, 8), (1100, 40, 8), (300, 4096, 32), (9000, 3, 1)])
def test_more_pairs_than_the_grouping_keeps(tokens, experts, top_k):
    """Up to 8192 pairs are put in order in shared memory; each token as in a call of its own."""
    gate_up, down = layer(128, 16, experts)
    x, ids, weights = batch(tokens, 128, experts, top_k)
    out = RoutedExperts(gate_up, down, top_k, tokens)(x, ids, weights)
    part = RoutedExperts(gate_up, down, top_k, 50)
    for start in (0, tokens // 2, tokens - 50):
        rows = slice(start, start + 50)
        assert torch.equal(out[rows], part(x[rows], ids[rows], weights[rows]))
    check(gate_up, down, x[-40:], ids[-40:], weights[-40:])


def test_as_an_opaque_operator():
    from cfm_b200.runtime import ops

    gate_up, down = layer(256, 48, 4)
    x, ids, weights = batch(20, 256, 4, 2)
    run = RoutedExperts(gate_up, down, 2, 20)
    out = torch.empty_like(x)
    torch.ops.cfm_b200.reader_forward(x, ids, weights, None, out, ops.register_reader(run))
    assert torch.equal(out, run(x, ids, weights))


def test_beside_the_reader_that_keeps_all_channels():
    """A reader that keeps every channel computes the same layer, from the same tensors."""
    from cfm_b200.reader.budget import compile_budget
    from cfm_b200.reader.progressive import ProgressiveReader

    gate_up, down = layer(256, 48, 4)
    x, ids, weights = batch(12, 256, 4, 2)
    plan = compile_budget(hidden_size=256, expert_width=48, top_k=2, retention=1.0, screen_keep=1.0)
    reader = ProgressiveReader(gate_up, down, None, None, plan, 12, selection_score="point")
    got, kept = RoutedExperts(gate_up, down, 2, 12)(x, ids, weights), reader(x, ids, weights)
    # The reader rounds gate, up, their product twice and each expert's sum to BF16.
    assert (got.float() - kept.float()).norm() < 0.02 * kept.float().norm()


def test_two_calls_at_once_with_workspaces_of_their_own():
    gate_up, down = layer(512, 96, 8)
    runs = [RoutedExperts(gate_up, down, 2, 200) for _ in range(2)]
    inputs = [batch(tokens, 512, 8, 2, seed) for tokens, seed in ((200, 3), (90, 4))]
    want = [run(*given) for run, given in zip(runs, inputs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(10):
        got = []
        for stream, run, given in zip(streams, runs, inputs):
            with torch.cuda.stream(stream):
                got.append(run(*given))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_decode_step_from_router_to_scores():
    """Router, layer, head and scores as one captured step, against the same in 64 bits."""
    hidden, experts, vocabulary = 512, 16, 5003
    gate_up, down = layer(hidden, 96, experts)
    x, _, _ = batch(9, hidden, experts, 4)
    generator = torch.Generator(device="cuda").manual_seed(4)
    router = 0.05 * torch.randn((experts, hidden), device="cuda", generator=generator)
    head = 0.05 * torch.randn((vocabulary, hidden), device="cuda", generator=generator)
    run = RoutedExperts(gate_up, down, 4, 9)
    tokens = torch.randint(0, vocabulary, (9,), device="cuda", generator=generator)
    before = x.float() @ head.T

    def step():
        weights, ids = route_tokens(x.float() @ router.T, 4)
        after = (x.float() + run(x, ids, weights).float()) @ head.T
        return weights, ids, after, token_logprobs(after, tokens, 5), compare_logits(before, after)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        weights, ids, after, scores, (divergence, agreement) = step()
    graph.replay()
    check(gate_up, down, x, ids, weights, run=run)
    log_p = torch.log_softmax(after.double(), -1)
    torch.testing.assert_close(scores.logprobs.double(), log_p.gather(1, tokens[:, None])[:, 0], rtol=1e-5, atol=1e-5)
    log_r = torch.log_softmax(before.double(), -1)
    torch.testing.assert_close(divergence.double(), (log_r.exp() * (log_r - log_p)).sum(-1), rtol=1e-5, atol=1e-7)
    assert torch.equal(agreement, before.argmax(-1) == after.argmax(-1))
    assert torch.equal(scores.top_ids[:, 0].long(), after.argmax(-1))


def test_refusals():
    gate_up, down = layer(256, 48, 4)
    for g, d in ((gate_up.float(), down), (gate_up, down.contiguous()), (gate_up, down[:3]),
                 (gate_up[:, :95], down), (gate_up[:, :, :128], down), (gate_up.cpu(), down.cpu()),
                 (gate_up[:, :, :250].contiguous(), channel_major_down(down[:, :250])),
                 (gate_up[:, :80].contiguous(), channel_major_down(down[:, :, :40])), (gate_up[0], down)):
        with pytest.raises(ValueError):
            RoutedExperts(g, d, 2, 8)
    for top_k, tokens in ((0, 8), (33, 8), (2, 0), (2, -1)):
        with pytest.raises(ValueError):
            RoutedExperts(gate_up, down, top_k, tokens)
    with pytest.raises(ValueError):
        RoutedExperts(gate_up, down, 2, 8, activation="relu")
    with pytest.raises(ValueError):
        RoutedExperts(gate_up, down, 2, 8, workspace=RoutedWorkspace(256, 48, 4, 3, 8, "cuda"))
    with pytest.raises(ValueError):
        RoutedExperts(gate_up, down, 2, 8, workspace=RoutedWorkspace(256, 48, 4, 2, 7, "cuda"))
    with pytest.raises(ValueError):
        RoutedExperts(gate_up, down, 2, 0, workspace=RoutedWorkspace(256, 48, 4, 2, 7, "cuda"))
    run = RoutedExperts(gate_up, down, 2, 8)
    x, ids, weights = batch(8, 256, 4, 2)
    for call in (
        (x[:0], ids[:0], weights[:0]), (torch.cat((x, x)), torch.cat((ids, ids)), torch.cat((weights, weights))),
        (x.float(), ids, weights), (x[:, :128], ids, weights), (x.cpu(), ids, weights), (x, ids.short(), weights),
        (x, ids, weights.half()), (x, ids[:7], weights[:7]), (x, ids[:, :1], weights[:, :1]), (x, ids, weights.T),
        (x, ids, weights, torch.zeros(7, device="cuda", dtype=torch.bool)),
        (x, ids, weights, torch.zeros(8, device="cuda", dtype=torch.uint8)),
        (x, ids, weights, None, torch.empty_like(x, dtype=torch.float32)),
        (x, ids, weights, None, torch.empty((8, 512), device="cuda", dtype=torch.bfloat16)[:, :256]),
        (x[0], ids, weights),
    ):
        with pytest.raises(ValueError):
            run(*call)
    wants = weights.clone().requires_grad_()
    with pytest.raises(ValueError, match="grad"):
        run(x, ids, wants)
    with torch.no_grad():
        run(x, ids, wants)
