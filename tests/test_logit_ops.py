"""Operators on rows of logits (logit_cases.py): on the device (marked gpu), and from the same sources on the host model
of the kernels (CPU suite), there also with the lanes taken in adverse orders."""
import numpy as np
import pytest
import torch

import emu_lib
import logit_cases as cases
from test_emulated_kernels import E   # noqa: F401  (fixture: the host build)

# vocabulary, bf16, padding of the rows: a wave, four waves and sixteen waves per row, sizes around a vector, odd ones
SHAPES = [(1, False, 0), (1, True, 3), (5, True, 0), (7, False, 2), (16, True, 0), (50, False, 0), (257, True, 0),
          (1000, False, 24), (2047, False, 0), (2051, False, 0), (2999, False, 5), (4099, True, 0), (4096, True, 8),
          (7003, True, 1), (9001, False, 1),
          (30522, True, 0), (30522, False, 6), (70001, False, 0), (140001, True, 0)]
ON_HOST = [s for s in SHAPES if s[0] < 10000]


def device_backend():
    from sfb import sfb

    def dev(a, bf16=False):
        t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
        return t.to(torch.bfloat16) if bf16 else t
    return sfb, dev


def host_backend(E, **how):
    emu_lib.configure(**how)
    return E, emu_lib.tensor


def top_of(vocab):
    return min(vocab, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", SHAPES)
def test_token_logprobs_on_the_device(vocab, bf16, pad):
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=1, k=top_of(vocab), repeat=2)
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=5, k=min(vocab, 64), scale=0.7, seed=3)
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=1, k=1, scale=1.6, seed=4, entropy=False)
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=20, k=min(vocab, 7), seed=6)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", SHAPES)
def test_token_logprobs_backward_on_the_device(vocab, bf16, pad):
    cases.logprobs_backward(*device_backend(), vocab, bf16, pad, n=1)
    cases.logprobs_backward(*device_backend(), vocab, bf16, pad, n=7, scale=0.6, entropy=False, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", SHAPES)
def test_distillation_on_the_device(vocab, bf16, pad):
    cases.distillation(*device_backend(), vocab, bf16, pad, slots=1)
    cases.distillation(*device_backend(), vocab, bf16, pad, slots=37, teacher_bf16=True, in_place=True, seed=11)
    cases.distillation(*device_backend(), vocab, bf16, pad, slots=256, scale=1.5, seed=12)


CUT = [(9001, False, 1), (30522, True, 0), (70001, False, 0), (140001, True, 0)]   # rows long enough to be cut


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", CUT)
def test_few_long_rows_cut_over_the_device(vocab, bf16, pad):
    S, dev = device_backend()
    ws = torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    for n, k in ((1, 20), (5, 64), (3, 0), (1, 1)):
        cases.logprobs(S, dev, vocab, bf16, pad, n=n, k=k, workspace=ws, repeat=3, seed=20 + k)
        for kind in ("normal", "masked", "nan"):   # one row: the most parts
            cases.logprobs(S, dev, vocab, bf16, pad, n=n, k=k, workspace=ws, kinds=[kind], seed=40 + k)
    for slots, teacher_bf16, in_place in ((1, False, False), (37, True, True), (256, False, False)):
        cases.distillation(S, dev, vocab, bf16, pad, slots=slots, teacher_bf16=teacher_bf16, in_place=in_place, workspace=ws, seed=30 + slots)
    torch.cuda.synchronize()
    assert int(ws[:2048].view(torch.int32).abs().sum()) == 0, "arrival counters must be left at zero"


# the same token several times, and tokens that the search for those cannot tell apart at first
@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16", [(3, False), (700, True), (2999, False), (30522, True), (70001, False), (140001, True)])
def test_few_tokens_named_many_times_on_the_device(vocab, bf16):
    for n in (2, 67, 256):
        cases.logprobs_backward(*device_backend(), vocab, bf16, 0, n=n, few=True, seed=70 + n)
        cases.distillation(*device_backend(), vocab, bf16, 1, slots=n, few=True, seed=71 + n)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16", [(70, False), (365, False), (1000, True), (2000, False), (3500, False), (9001, True), (30522, False), (140001, True)])
def test_alternatives_behind_masks_and_among_ties_on_the_device(vocab, bf16):
    S, dev = device_backend()
    ws = torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    for k in (1, 20, 33, 64):
        cases.logprobs(S, dev, vocab, bf16, 0, n=1, k=k, kinds=cases.MASKS_AND_TIES, seed=90 + k)
        cases.logprobs(S, dev, vocab, bf16, 3, n=1, k=k, kinds=cases.MASKS_AND_TIES, seed=91 + k, workspace=ws, repeat=2)


CLUSTERED = ["rising", "falling", "first ones large", "coarse", "nan", "inf"]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16", [(70, False), (1000, True), (2999, False), (8190, True), (9001, False), (40000, True), (70001, False), (131072, False)])
def test_clustered_alternatives_on_the_device(vocab, bf16):
    S, dev = device_backend()
    ws = torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    for k in (9, 16, 17, 32, 33, 64):
        cases.logprobs(S, dev, vocab, bf16, 1, n=1, k=k, kinds=CLUSTERED, seed=160 + k, repeat=2)
        cases.logprobs(S, dev, vocab, bf16, 0, n=1, k=k, kinds=CLUSTERED, seed=161 + k, repeat=2, workspace=ws)


# the kernels a distillation's loss and gradient come from in one launch, by the largest number of 16-byte vectors in a row
GRADIENT_SHAPES = [(64, "64, 1"), (256, "64, 4"), (512, "64, 8"), (1024, "128, 8"), (2048, "256, 8"), (4096, "512, 8"),
                   (8192, "512, 16"), (12288, "512, 24"), (16384, "1024, 16"), (20000, "1024, 0")]


def at_the_limit(vecs, bf16, over):
    """The odd vocabulary closest to the limit that still is (over: no longer is) within it."""
    n = 8 if bf16 else 4
    return vecs * n + (n + 1 if over else n - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("vecs", [vecs for vecs, _ in GRADIENT_SHAPES])
def test_every_shape_of_the_distillation_gradient_on_the_device(vecs, bf16):
    for over in (False, True):
        vocab = at_the_limit(vecs, bf16, over)
        cases.distillation(*device_backend(), vocab, bf16, 0, slots=9, seed=150)
        cases.distillation(*device_backend(), vocab, bf16, 0, slots=130, teacher_bf16=True, in_place=True, seed=151, few=True)


FAR_APART = [(11, False), (200, True), (1000, False), (2500, False), (9001, True), (40000, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16", FAR_APART)
def test_logits_far_apart_on_the_device(vocab, bf16):
    S, dev = device_backend()
    cases.far_apart(S, dev, vocab, bf16)
    cases.far_apart(S, dev, vocab, bf16, workspace=torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda"))


# masks whose scaled value is -1e30 in fp32 (the products' factors are 1 and 10), or close to it
FAR_MASKS = [(-1e30, float(np.float32(np.log(2.0)))), (-1e29, 6.931472)]


@pytest.mark.gpu
@pytest.mark.parametrize("mask,scale", FAR_MASKS)
@pytest.mark.parametrize("vocab,bf16", [(300, True), (9001, False), (20000, True), (70001, False), (140001, True)])
def test_far_masks_on_the_device(vocab, bf16, mask, scale):
    S, dev = device_backend()
    cases.far_masks(S, dev, vocab, bf16, mask, scale)
    cases.far_masks(S, dev, vocab, bf16, mask, scale, workspace=torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda"))


FAR_FROM_ZERO = [(-1e10, 1.0), (-3e10, 0.7), (-1e20, 1.0), (-1e29, 1.0), (1e10, 1.0), (-2.0 ** 24, 1.0), (-3e7, 0.7), (-1e10, 1e-3)]


@pytest.mark.gpu
@pytest.mark.parametrize("value,scale", FAR_FROM_ZERO)
@pytest.mark.parametrize("vocab,bf16", [(200, False), (3000, False), (9001, False), (20000, True), (140001, True)])
def test_logits_far_from_zero_on_the_device(vocab, bf16, value, scale):
    S, dev = device_backend()
    cases.far_from_zero(S, dev, vocab, bf16, value, scale)
    cases.far_from_zero(S, dev, vocab, bf16, value, scale, workspace=torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda"))


LARGE_WEIGHTS = [(1e-4, 1e33), (1e-3, 5e33)]


@pytest.mark.gpu
@pytest.mark.parametrize("scale,weight", LARGE_WEIGHTS)
@pytest.mark.parametrize("vocab,bf16", [(300, True), (3000, False), (9001, False), (70001, False), (140001, True)])
def test_large_weights_on_the_device(vocab, bf16, scale, weight):
    S, dev = device_backend()
    cases.large_weights(S, dev, vocab, bf16, scale, weight)
    cases.large_weights(S, dev, vocab, bf16, scale, weight, workspace=torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda"))


@pytest.mark.gpu
def test_teacher_to_student_on_the_device():
    cases.teacher_to_student(*device_backend())


@pytest.mark.gpu
def test_parts_left_out_on_the_device():
    cases.parts_left_out(*device_backend())


@pytest.mark.gpu
def test_rows_far_apart_on_the_device():
    cases.one_row_of_many(*device_backend())
    cases.one_row_of_many(*device_backend(), rows=3)


@pytest.mark.gpu
@pytest.mark.needs_device
def test_host_tensors_are_refused():
    S, dev = device_backend()
    x = dev(np.zeros((2, 40), np.float32))
    tok = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: S.token_logprobs(x, tok), lambda: S.token_logprobs(x.cpu(), tok), lambda: S.distillation_loss(x, tok[:, None], x[:, :1].cpu())):
        with pytest.raises(S.SfbError) as e:
            call()
        assert e.value.status == 8


@pytest.mark.gpu
@pytest.mark.needs_device
def test_on_another_stream():
    S, dev = device_backend()
    x = dev(cases.matrix(30522, 3, False, ["normal"] * 40))
    tok = torch.arange(40, dtype=torch.int32, device="cuda")
    want = S.token_logprobs(x, tok, top_k=8, entropy=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = S.token_logprobs(x, tok, top_k=8, entropy=True)
        d = S.token_logprobs_backward(x, tok, got["stats"], d_logprob=got["logprob"])
    side.synchronize()
    for name in want:
        assert torch.equal(got[name], want[name]), name
    assert torch.equal(d, S.token_logprobs_backward(x, tok, want["stats"], d_logprob=want["logprob"]))


@pytest.mark.gpu
@pytest.mark.needs_device
def test_captured_and_replayed_with_a_shared_workspace():
    """Two graphs with one workspace, replayed in turn on changing inputs with eager calls between: every replay gives
    what the eager call gives."""
    S, dev = device_backend()
    ws = torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(5)
    few, many = torch.empty((3, 70001), device="cuda"), torch.empty((900, 5003), device="cuda", dtype=torch.bfloat16)
    tok = dev(rng.integers(0, 5003, 900).astype(np.int32))
    ids, z = dev(rng.integers(0, 5003, (900, 17)).astype(np.int32)), dev(rng.standard_normal((900, 17)).astype(np.float32))
    w = dev(rng.standard_normal(900).astype(np.float32))

    def first():
        a = S.token_logprobs(few, tok[:3], top_k=20, entropy=True, workspace=ws)
        b = S.distillation_loss(few, ids[:3], z[:3], scale=0.5, d_loss=w[:3], workspace=ws)
        return [a[n] for n in sorted(a)] + [b[n] for n in sorted(b)]

    def second():
        a = S.token_logprobs(many, tok, top_k=5, entropy=True, workspace=ws)
        d = S.token_logprobs_backward(many, tok, a["stats"], d_logprob=w, entropy=a["entropy"], d_entropy=w)
        b = S.distillation_loss(many, ids, z, scale=0.5, d_loss=w, workspace=ws)
        c = S.distillation_loss(few, ids[:3], z[:3], workspace=ws)
        return [a[n] for n in sorted(a)] + [b[n] for n in sorted(b)] + [c["row_loss"], d]

    few.normal_()
    many.normal_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first(), second()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for call in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out, call))
    for turn in range(4):
        few.normal_(0, 1 + turn)
        many.normal_(0, 1 + turn)
        for g, out, call in graphs:
            g.replay()
            torch.cuda.synchronize()
            for got, want in zip(out, call()):
                assert torch.equal(got, want)
    assert int(ws[:2048].view(torch.int32).abs().sum()) == 0


@pytest.mark.gpu
@pytest.mark.needs_device
def test_offsets_past_32_bits():
    """Rows that begin more than 2^32 elements (and 2^33 bytes) into the logits."""
    S, _ = device_backend()
    rows, vocab = 70000, 65541
    x = torch.empty((rows, vocab), device="cuda", dtype=torch.bfloat16)
    x.zero_()
    x[-3:].normal_(0, 2)
    x[0].normal_(0, 2)
    tok = torch.full((rows,), 65540, device="cuda", dtype=torch.int32)
    some = torch.tensor([0, rows - 3, rows - 2, rows - 1], device="cuda")
    got = S.token_logprobs(x, tok, entropy=True)
    lp = torch.log_softmax(x[some].double(), 1)
    assert (got["logprob"][some].double() - lp[:, -1]).abs().max() < 2e-5
    assert abs(float(got["logprob"][5]) + np.log(vocab)) < 2e-5 and abs(float(got["entropy"][5]) - np.log(vocab)) < 2e-4
    g = torch.zeros(rows, device="cuda")
    g[some] = 1.0
    d = S.token_logprobs_backward(x, tok, got["stats"], d_logprob=g, out=x)
    want = -lp.exp()
    want[:, -1] += 1
    assert (d[some].double() - want).abs().max() < 2.0 ** -8 * 1.01
    assert not d[1:rows - 3:9999].any()
    assert int((d[1:rows - 3] != 0).sum()) == 0


@pytest.mark.gpu
def test_model_scores_its_input():
    """Model.score: the log probabilities of given tokens are minus the losses the model's own cross-entropy gives; the
    best alternatives are its largest logits."""
    S, dev = device_backend()
    rng = np.random.default_rng(9)
    bs, nb, heads, d, vocab, ffn = 64, 4, 2, 64, 500, 128
    n, L = heads * d, bs * nb
    f32 = lambda *shape: dev((rng.standard_normal(shape) * 0.05).astype(np.float32))   # noqa: E731
    w = {name: f32(*shape) for name, shape in (("wq", (n, n)), ("wk", (n, n)), ("wv", (n, n)), ("wo", (n, n)), ("w1", (n, ffn)), ("w2", (ffn, n)),
                                               ("bq", (n,)), ("bk", (n,)), ("bv", (n,)), ("bo", (n,)), ("b1", (ffn,)), ("b2", (n,)),
                                               ("ln1_b", (n,)), ("ln2_b", (n,)))}
    w["ln1_g"], w["ln2_g"] = (dev(np.ones(n, np.float32)) for _ in range(2))
    model = S.Model(f32(vocab, n), f32(L, n), [w], S.build_luts(S.layout_local(nb, 1, bidirectional=True)), bs, heads, d, ffn)
    ids = dev(rng.integers(0, vocab, (2, L)).astype(np.int32))
    labels = dev(rng.integers(0, vocab, (2, L)).astype(np.int32))
    logits = model.forward(ids, want_logits=True)["logits"]
    _, row_loss = S.softmax_cross_entropy(logits, labels.reshape(-1))
    got = model.score(ids, labels, top_k=10, entropy=True)
    assert np.abs(cases.host(got["logprob"]) + cases.host(row_loss)).max() < 1e-5
    assert np.array_equal(cases.host(got["top_ids"]), cases.plain_top(cases.host(logits).astype(np.float32), 10))
    pair = torch.stack([labels, ids], dim=2).contiguous()
    assert torch.equal(model.score(ids, pair)["logprob"][:, 0], got["logprob"])
    with pytest.raises(S.SfbError):
        model.score(ids, labels[:1])


@pytest.mark.gpu
def test_refusals_on_the_device():
    cases.refusals(*device_backend())


@pytest.mark.parametrize("vocab,bf16,pad", ON_HOST)
def test_token_logprobs_on_the_host_model(E, vocab, bf16, pad):   # noqa: F811
    cases.logprobs(*host_backend(E), vocab, bf16, pad, n=1, k=top_of(vocab))
    cases.logprobs(*host_backend(E), vocab, bf16, pad, n=5, k=min(vocab, 64), scale=0.7, seed=3)
    cases.logprobs(*host_backend(E), vocab, bf16, pad, n=20, k=min(vocab, 7), seed=6)


@pytest.mark.parametrize("vocab,bf16,pad", ON_HOST)
def test_token_logprobs_backward_on_the_host_model(E, vocab, bf16, pad):   # noqa: F811
    cases.logprobs_backward(*host_backend(E), vocab, bf16, pad, n=1)
    cases.logprobs_backward(*host_backend(E), vocab, bf16, pad, n=7, scale=0.6, entropy=False, in_place=True)


@pytest.mark.parametrize("vocab,bf16,pad", ON_HOST)
def test_distillation_on_the_host_model(E, vocab, bf16, pad):   # noqa: F811
    cases.distillation(*host_backend(E), vocab, bf16, pad, slots=1)
    cases.distillation(*host_backend(E), vocab, bf16, pad, slots=37, teacher_bf16=True, in_place=True, seed=11)


@pytest.mark.parametrize("vocab,bf16,order", [(8200, False, 0), (9001, False, 14), (16400, True, 1), (25003, True, 21)])
def test_few_long_rows_cut_on_the_host_model(E, vocab, bf16, order):   # noqa: F811
    S, dev = host_backend(E, order=order)
    ws = dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8))
    cases.logprobs(S, dev, vocab, bf16, 3, n=5, k=9, workspace=ws, kinds=["normal", "masked", "rising", "nan", "all lowest", "empty"], repeat=2)
    cases.logprobs(S, dev, vocab, bf16, 0, n=1, k=64, workspace=ws, kinds=["ties"], seed=8)
    cases.distillation(S, dev, vocab, bf16, 0, slots=37, workspace=ws, kinds=["normal", "masked", "rising", "empty", "nan", "late peak"], in_place=True)
    assert not ws[:2048].any(), "arrival counters must be left at zero"


@pytest.mark.parametrize("order", [1, 14, 21])
def test_logit_ops_with_lanes_in_adverse_orders(E, order):   # noqa: F811
    back = host_backend(E, order=order)
    cases.logprobs(*back, 2500, False, 1, n=5, k=40)
    cases.logprobs_backward(*back, 2500, False, 1, n=5, in_place=True)
    cases.distillation(*back, 4200, True, 3, slots=70, in_place=True)
    cases.distillation(*back, 900, False, 0, slots=70, in_place=True)


@pytest.mark.parametrize("vocab,bf16", [(2100, False), (3500, False), (4099, False), (4200, True), (8190, True)])
def test_a_wave_ahead_of_the_others_among_many_alternatives(E, vocab, bf16):   # noqa: F811
    """Rows of two waves whose lists of alternatives are long enough to be thinned out: whichever wave is ahead, all of
    them come to every barrier."""
    for order in (-1, -2):
        S, dev = host_backend(E, order=order)
        E.lib.emu_reset_counts()
        for k in (33, 64):
            cases.logprobs(S, dev, vocab, bf16, 0, n=1, k=k, kinds=["rising", "normal", "ties", "rising", "spread ties"], seed=130 + k)
        whole, missed = emu_lib.counts()["block_barrier"]
        assert whole and missed == 0, (order, missed)
    emu_lib.configure()


@pytest.mark.parametrize("vocab,bf16", [(2999, False), (8190, True), (9001, False), (40000, True), (70001, False)])
def test_reads_of_rows_with_clustered_alternatives(E, vocab, bf16):   # noqa: F811
    """However the largest logits stand together, a row is read a bounded number of times, not once for every bit of a
    logit: the work-group meets four times for each read, and twice for every step that looks for equal logits."""
    vecs = vocab // (8 if bf16 else 4)
    steps = -(-vocab // (128 if vecs <= 1024 else 256 if vecs <= 4096 else 512))
    S, dev = host_backend(E)
    tok = dev(np.zeros(1, np.int32))
    for kind in CLUSTERED:
        x = dev(cases.matrix(vocab, 7, bf16, [kind]), bf16)
        for k in (9, 16, 17, 20, 32, 33, 64):
            E.lib.emu_reset_counts()
            S.token_logprobs(x, tok, top_k=k)
            assert emu_lib.counts()["block_barrier"][0] < 4 * 10 + 2 * steps, (kind, k)
    for k in (9, 17, 64):
        cases.logprobs(S, dev, vocab, bf16, 1, n=1, k=k, kinds=CLUSTERED, seed=160 + k)
        cases.logprobs(S, dev, vocab, bf16, 0, n=1, k=k, kinds=CLUSTERED, seed=161 + k, workspace=dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8)))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("at", range(len(GRADIENT_SHAPES)))
def test_every_shape_of_the_distillation_gradient_on_the_host_model(E, at, bf16):   # noqa: F811
    S, dev = host_backend(E)
    vecs, shape = GRADIENT_SHAPES[at]
    some = ["normal", "lowest", "ties", "late peak", "masked", "peaked", "normal"]
    for over in (False, True):
        expected = shape if not over else GRADIENT_SHAPES[min(at + 1, len(GRADIENT_SHAPES) - 1)][1]
        vocab = at_the_limit(vecs, bf16, over)
        E.lib.emu_reset_counts()
        S.distillation_loss(dev(cases.matrix(vocab, 1, bf16, ["normal"]), bf16), dev(np.zeros((1, 3), np.int32)), dev(np.zeros((1, 3), np.float32)),
                            d_loss=dev(np.ones(1, np.float32)))
        # (the two the sources write out: with the gradient only, and with the loss alone too)
        assert len(emu_lib.launched()) == 1 and emu_lib.launched() <= {"distill_kernel<T, %s, %s>" % (expected, g) for g in ("GRAD", "true")}
        cases.distillation(S, dev, vocab, bf16, 0, slots=9, seed=150, kinds=some)
        cases.distillation(S, dev, vocab, bf16, 0, slots=130, teacher_bf16=True, in_place=True, seed=151, few=True, kinds=some)


@pytest.mark.parametrize("vocab,bf16,order", [(3, False, 0), (700, True, 14), (2999, False, 1), (9001, True, 0)])
def test_few_tokens_named_many_times_on_the_host_model(E, vocab, bf16, order):   # noqa: F811
    back = host_backend(E, order=order)
    some = ["normal", "masked", "nan", "lowest", "empty"]
    for n in (2, 67):
        cases.logprobs_backward(*back, vocab, bf16, 0, n=n, few=True, seed=70 + n, kinds=some)
        cases.distillation(*back, vocab, bf16, 1, slots=n, few=True, seed=71 + n, kinds=some)


@pytest.mark.parametrize("vocab,bf16,order", [(70, False, 0), (365, False, 1), (2000, False, 14), (3500, False, 0), (9001, True, 21)])
def test_alternatives_behind_masks_and_among_ties_on_the_host_model(E, vocab, bf16, order):   # noqa: F811
    S, dev = host_backend(E, order=order)
    ws = dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8))
    for k in (20, 64):
        cases.logprobs(S, dev, vocab, bf16, 3, n=1, k=k, kinds=cases.MASKS_AND_TIES, seed=90 + k)
        cases.logprobs(S, dev, vocab, bf16, 0, n=1, k=k, kinds=cases.MASKS_AND_TIES, seed=91 + k, workspace=ws)


@pytest.mark.parametrize("vocab,bf16", FAR_APART[:-1])
def test_logits_far_apart_on_the_host_model(E, vocab, bf16):   # noqa: F811
    S, dev = host_backend(E)
    cases.far_apart(S, dev, vocab, bf16)
    cases.far_apart(S, dev, vocab, bf16, workspace=dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8)))


@pytest.mark.parametrize("mask,scale", FAR_MASKS)
@pytest.mark.parametrize("vocab,bf16", [(300, True), (3000, False), (9001, False), (20000, True)])
def test_far_masks_on_the_host_model(E, vocab, bf16, mask, scale):   # noqa: F811
    S, dev = host_backend(E)
    cases.far_masks(S, dev, vocab, bf16, mask, scale)
    cases.far_masks(S, dev, vocab, bf16, mask, scale, workspace=dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8)))


@pytest.mark.parametrize("value,scale", FAR_FROM_ZERO)
@pytest.mark.parametrize("vocab,bf16", [(200, False), (3000, False), (9001, False), (20000, True)])
def test_logits_far_from_zero_on_the_host_model(E, vocab, bf16, value, scale):   # noqa: F811
    S, dev = host_backend(E)
    cases.far_from_zero(S, dev, vocab, bf16, value, scale, workspace=dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8)) if vocab > 9000 else None)


@pytest.mark.parametrize("scale,weight", LARGE_WEIGHTS)
@pytest.mark.parametrize("vocab,bf16", [(300, True), (3000, False), (9001, False), (70001, False)])
def test_large_weights_on_the_host_model(E, vocab, bf16, scale, weight):   # noqa: F811
    S, dev = host_backend(E)
    cases.large_weights(S, dev, vocab, bf16, scale, weight, workspace=dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8)) if vocab > 9000 else None)


def test_teacher_to_student_on_the_host_model(E):   # noqa: F811
    cases.teacher_to_student(*host_backend(E))


def test_parts_left_out_on_the_host_model(E):   # noqa: F811
    cases.parts_left_out(*host_backend(E))


def test_rows_far_apart_on_the_host_model(E):   # noqa: F811
    cases.one_row_of_many(*host_backend(E))
    cases.one_row_of_many(*host_backend(E), rows=3)


def test_refusals_on_the_host_model(E):   # noqa: F811
    cases.refusals(*host_backend(E))
