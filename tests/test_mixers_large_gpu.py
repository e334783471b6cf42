"""gpu: the paths that large calls of the mixers take, at sizes that follow the number of SMs: runs of several groups of rows, wide scans of more blocks
than there are SMs, several rows of a batch in a block, attention rows beyond one chunk of masks."""
import pytest
import torch

import causal_flare as cf
from oracle import mixers_oracle as orc
from test_attention_gpu import behind_a_cache, close as attention_close
from test_state_space_gpu import close, gen, ids, magnitudes, near, randn, scan_inputs

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", [None, "holes"])
def test_conv_runs_of_several_groups(kind, dtype):
    # blocks enough along batch and channels for the places of all SMs (six blocks each, of 128 channels): a row is four runs of 32 tokens, of four groups
    # of eight rows, the last run cut off in its first
    C, N, W = 1024, 101, 4
    B = sms() * 6 // (C // 128) + 1
    g = gen(21)
    x, w, bias, dy = randn(g, B, N, C, dtype=dtype), randn(g, C, W), randn(g, C), randn(g, B, N, C, dtype=dtype)
    docs = ids(kind, B, N, g)
    leaves = [x, w, bias]
    for t in leaves:
        t.requires_grad_()
    y = cf.flare_causal_conv(x, w, bias, activation="silu", documents=docs)
    got = torch.autograd.grad(y, leaves, dy)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    want = orc.causal_conv(*exact, silu=True, documents=docs)[0]
    grads = torch.autograd.grad(want, exact, dy.double())
    size = orc.causal_conv(*(t.detach().double().abs() for t in leaves), documents=docs)[0]
    close(y, want.detach(), size, W, "y")
    for name, a, b, t in zip(("dx", "dw", "dbias"), got, grads, (dtype, torch.float32, torch.float32)):
        near(a, b, t, W, name)
    if kind is None:  # the same rows behind a state
        state = randn(g, B, W - 1, C, dtype=dtype)
        lengths = torch.randint(0, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        with torch.no_grad():
            y, out = cf.flare_causal_conv_prefill(x, w, bias, state, activation="silu", lengths=lengths)
            want, left = orc.causal_conv(*exact, state.double(), True, lengths=lengths)
            size = orc.causal_conv(*(t.double().abs() for t in leaves), state.double().abs(), lengths=lengths)[0]
        close(y, want, size, W, "prompt")
        assert torch.equal(out.double(), left)


def scan_case(name):
    blocks = sms() + 1
    if name == "batch":  # more blocks than SMs by batch and channels alone: one segment
        return -(-blocks // 8), 70, 512
    if name == "segments":  # one block of channels, eight segments and more
        return 1, 1200, 64
    return 1, -(-blocks // 5) * 128 + 9, 320  # segments of four tiles, more blocks than SMs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name, kind", [("batch", None), ("batch", "holes"), ("segments", None), ("segments", "again"), ("both", "some")])
def test_scans_of_many_blocks(name, kind, dtype):
    B, N, C = scan_case(name)
    g = gen(22)
    t = scan_inputs(g, B, N, C, 16, 1, dtype)
    docs = ids(kind, B, N, g)
    if kind == "some":  # (documents that are longer than a segment)
        docs = torch.arange(N, device="cuda")[None].repeat(B, 1).int() // 700
    dy = randn(g, B, N, C, dtype=dtype)
    for v in t.values():
        v.requires_grad_()
    y = cf.flare_selective_scan(**t, dt_softplus=True, documents=docs)
    got = torch.autograd.grad(y, list(t.values()), dy)
    exact = {k: v.detach().double().requires_grad_() for k, v in t.items()}
    want = orc.selective_scan(**exact, softplus=True, documents=docs)[0]
    grads = torch.autograd.grad(want, list(exact.values()), dy.double())
    with torch.no_grad():
        size = magnitudes({k: v.detach() for k, v in t.items()}, softplus=True, documents=docs)[0]
    close(y, want.detach(), size, N, "y")
    for (which, v), a, b in zip(t.items(), got, grads):
        near(a, b, v.dtype, N, which)


@pytest.mark.parametrize("S", [8, 16, 32])
def test_long_prompts_of_many_blocks(S):
    B, N, C = scan_case("both")
    g = gen(23 + S)
    with torch.no_grad():
        t = scan_inputs(g, B, N, C, S, 1, torch.bfloat16)
        state, lengths = randn(g, B, C, S), torch.tensor([N - 133], device="cuda", dtype=torch.int32)
        y, out = cf.flare_selective_scan_prefill(**t, state=state, dt_softplus=True, lengths=lengths)
        want, left = orc.selective_scan(**{k: v.double() for k, v in t.items()}, state=state.double(), softplus=True, lengths=lengths)
        ys, hs = magnitudes(t, state=state.double().abs(), softplus=True, lengths=lengths)
    close(y, want, ys, N, "y")
    close(out, left, hs, N, "state")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("S", [8, 16, 32])
def test_single_tokens_of_large_batches(S, dtype):
    # two blocks for every SM at four rows a block, and a last block of three
    B, C = 4 * 2 * sms() + 3, 200
    g = gen(24)
    t = scan_inputs(g, B, 1, C, S, 1, dtype, lead=(B,))
    state = randn(g, B, C, S)
    before = state.double()
    y, same = cf.flare_selective_scan_decode(**t, state=state, dt_softplus=True)
    assert same.data_ptr() == state.data_ptr()
    row = {k: (v[:, None] if k in ("x", "dt", "z", "B", "C") else v) for k, v in t.items()}
    want, left = orc.selective_scan(**{k: v.double() for k, v in row.items()}, state=before, softplus=True)
    ys, hs = magnitudes(row, state=before.abs(), softplus=True)
    close(y, want[:, 0], ys[:, 0], 1, "y")
    close(state, left, hs, 1, "state")


@pytest.mark.parametrize("case", ["documents", "prefix", "window"])
def test_attention_rows_beyond_a_chunk_of_masks(case):
    # 4 096 tokens are looked at together: documents and prefixes that lie across that border (and across the next), padding behind the first 32 tiles of 64
    B, N, H, J, D = 1, 4500 if case != "window" else 8300, 2, 1, 64
    g = gen(25)
    q, k, v = randn(g, B, N, H, D, dtype=torch.bfloat16), randn(g, B, N, J, D, dtype=torch.bfloat16), randn(g, B, N, J, D, dtype=torch.bfloat16)
    dy = randn(g, B, N, H, D, dtype=torch.bfloat16)
    at = torch.arange(N, device="cuda")[None]
    documents = prefix = window = None
    if case == "documents":
        documents = torch.where(at < 3700, at // 900, torch.where(at < 4400, 9, 10)).int()
        documents = torch.where((at > 2500) & (at < 2600) | (at > 4450), -1, documents).int()
        prefix = (at < 300) | (at >= 3700) & (at < 4250)
    elif case == "prefix":  # of one document, up to behind the border
        prefix = at < 4200
    else:
        window = 500
        documents = torch.where(at < 4000, 0, torch.where(at < 8250, 1, -1)).int()
    for t in (q, k, v):
        t.requires_grad_()
    y = cf.flare_causal_attention(q, k, v, documents=documents, prefix=prefix, window=window)
    got = torch.autograd.grad(y, (q, k, v), dy)
    with torch.no_grad():
        see = orc.in_sight(N, documents, prefix, window).cuda()
        for h in range(H):  # (a head at a time: the oracle's tables take gigabytes)
            o = orc.Attention(q[:, :, h:h + 1].double(), k.double(), v.double(), see, D ** -0.5, dy=dy[:, :, h:h + 1].double(), eps=2.0 ** -8)
            attention_close(y[:, :, h:h + 1], o.y, o.y_off, f"y of head {h}")
            attention_close(got[0][:, :, h:h + 1], o.dq, o.dq_off, f"dq of head {h}")
            sums = (o.dk, o.dk_off, o.dv, o.dv_off) if h == 0 else tuple(a + b for a, b in zip(sums, (o.dk, o.dk_off, o.dv, o.dv_off)))
    attention_close(got[1], sums[0], sums[1], "dk")
    attention_close(got[2], sums[2], sums[3], "dv")


def test_prompts_behind_long_caches():
    B, N, H, J, D, L = 3, 200, 2, 1, 128, 4700
    g = gen(26)
    q, k, v = randn(g, B, N, H, D, dtype=torch.float16), randn(g, B, N, J, D, dtype=torch.float16), randn(g, B, N, J, D, dtype=torch.float16)
    cached, lengths = torch.tensor([4500, 2100, 40], device="cuda", dtype=torch.int32), torch.tensor([200, 130, 200], device="cuda", dtype=torch.int32)
    kc, vc = randn(g, B, L, J, D, dtype=torch.float16), randn(g, B, L, J, D, dtype=torch.float16)
    for b in range(B):
        kc[b, cached[b]:], vc[b, cached[b]:] = float("nan"), float("inf")
    y = cf.flare_causal_attention_prefill(q, k, v, kc, vc, cached=cached, lengths=lengths)
    see = behind_a_cache(B, N, L, cached, lengths, None)
    o = orc.Attention(q.double(), kc.double().nan_to_num(0, 0, 0), vc.double().nan_to_num(0, 0, 0), see, D ** -0.5, first=cached, eps=2.0 ** -11)
    attention_close(y, o.y, o.y_off, "y")
