"""The paged attention stack as a server uses it: prompt slices into pages,
forks, decode steps over the shared prefix (eager and captured), copy on write,
release and compaction. Checked against the same stack on flat caches, fed
through the calls that tests/test_gpu_stack.py and tests/test_gpu_gqa.py pin.

Tolerance: the paged decode keeps more terms of q and of the softmax weights
than the flat one (whose fp32 outputs are within 6e-6 of the exact row, relative
to its 2-norm; the paged one's within 5e-6), so an attention layer's output
differs by 1.1e-5 at most; the out-projection and the recurrent layers pass a
relative difference on without growing it by more than their condition, for
which 10 is allowed: 1.1e-4 of the step's largest residual update. Prompt
slices of more than 128 tokens run the same kernels on the same rows: the same
bits. Shorter ones take the decode's kernels on pages, where the flat prefill's
fp16 operands leave 3e-4 of a row: with two attention layers and the same
allowance of 10, 6.1e-3 of the slice's largest update. The flat stack then goes
on from the paged one's state, so that the steps are compared by themselves."""
import pytest
import torch

from gpu_util import DEV
from qff import synth

pytestmark = pytest.mark.gpu

N_LAYERS, SLOTS, MAX_CTX, PAGE = 8, 6, 1024, 64


@pytest.fixture(scope="module")
def model(hip):
    import qff
    from qff import stack as S
    g = torch.Generator(device=DEV).manual_seed(77)
    dnp = {k: torch.from_numpy(v).to(DEV) for k, v in synth.deltanet_params().items()}
    gqp = {k: torch.from_numpy(v).to(DEV) for k, v in synth.gqa_params().items()}
    layers = S.random_layers(N_LAYERS, g, dnp, gqp, device=DEV)
    ctx = qff.Context(max_batch=SLOTS, max_ctx=MAX_CTX, max_prefill_tokens=512)
    yield ctx, layers
    ctx.close()


def _stacks(model, pages=40):
    from qff.pages import PageTable
    from qff.stack import AttentionStack
    ctx, layers = model
    table = PageTable(pages, PAGE, SLOTS, MAX_CTX, device=DEV)
    return AttentionStack(ctx, layers, SLOTS, MAX_CTX, pages=table), AttentionStack(ctx, layers, SLOTS, MAX_CTX)


def _flat_prefill(st, slot, x, start):
    """The slice through a flat stack's own calls."""
    from qff import ops
    T = x.shape[0]
    for kind, L, S in zip(st.kinds, st.layers, st.states):
        y = ops.q4_norm_matmul_parts(st.ctx, L["in_proj"], x, L["in_norm_w"], st.eps)
        if kind == "dn":
            core = ops.deltanet_prefill(st.ctx, L["params"], y[0], y[1], y[3], y[2], S["conv_state"][slot], S["ssm_state"][slot],
                                        out_dtype=torch.float32, eps=st.eps)
        else:
            core = ops.gqa_prefill(st.ctx, L["params"], y[0].view(T, 16, 512), y[1].view(T, 2, 256), y[2].view(T, 2, 256),
                                   S["k_cache"][slot], S["v_cache"][slot], start_pos=start, out_dtype=torch.float32,
                                   eps=st.eps).view(T, 4096)
        ops.q4_matmul_parts(st.ctx, [L["out_proj"]], core, outs=(x,), residuals=(x,))


def _prefill(paged, flat, slot, x, start):
    """A slice of both, compared; the flat one takes over the paged one's state."""
    a, b = x.clone(), x.clone()
    paged.prefill(slot, a, start)
    _flat_prefill(flat, slot, b, start)
    if x.shape[0] > 128:
        assert torch.equal(a, b)
    assert float((a - b).abs().max() / (b - x).abs().max()) <= 6.1e-3
    n = paged.pages.lengths[slot]
    at = paged.pages.table[slot, :-(-n // PAGE)].long()
    for kind, S, F in zip(paged.kinds, paged.states, flat.states):
        if kind == "gqa":
            F["k_cache"][slot, :n] = S["k_pages"][at].flatten(0, 1)[:n]
            F["v_cache"][slot, :n] = S["v_pages"][at].flatten(0, 1)[:n]
        else:
            F["conv_state"][slot], F["ssm_state"][slot] = S["conv_state"][slot], S["ssm_state"][slot]


def _flat_fork(st, src, dsts):
    for S in st.states:
        for t in S.values():
            for d in dsts:
                t[d] = t[src]


def _step(paged, flat, g, positions, graph=None):
    """One decode step of both; compares the active slots' residual updates."""
    x = torch.randn(SLOTS, 2048, device=DEV, generator=g)
    pos = torch.tensor(positions, dtype=torch.int32, device=DEV)
    a, b = x.clone(), x.clone()
    paged.reserve(positions)
    if graph is None:
        paged.decode_step(a, pos)
    else:
        graph["x"].copy_(x)
        graph["pos"].copy_(pos)
        graph["graph"].replay()
        torch.cuda.synchronize()
        a = graph["x"].clone()
    flat.decode_step(b, pos)
    on = [s for s, p in enumerate(positions) if p >= 0]
    da, db = (a - x)[on], (b - x)[on]
    assert not torch.isnan(da).any()
    assert float((da - db).abs().max() / db.abs().max()) <= 1.1e-4


def _same_cache(paged, flat, slots):
    """The rows that the slots hold, to what the decode steps may differ by (one
    step of bf16 of k, where its inputs differ in their last bits)."""
    P = paged.pages
    for kind, S, F in zip(paged.kinds, paged.states, flat.states):
        if kind != "gqa":
            continue
        for s in slots:
            n = P.lengths[s]
            at = P.table[s, :-(-n // PAGE)].long()
            for pool, cache in (("k_pages", "k_cache"), ("v_pages", "v_cache")):
                got = S[pool][at].flatten(0, 1)[:n].float()
                want = F[cache][s, :n].float()
                assert ((got - want).abs() <= 2.0 ** -6 * want.abs() + 1e-3).all(), (s, pool)


def test_prefill_then_decode(model):
    """Prompts of odd lengths in two slices into different slots, then steps."""
    paged, flat = _stacks(model)
    g = torch.Generator(device=DEV).manual_seed(1)
    lens = [137, 64, 0, 300, 1, 511]
    for s, n in enumerate(lens):
        at = 0
        for T in (n - n // 3, n // 3):
            if T:
                _prefill(paged, flat, s, torch.randn(T, 2048, device=DEV, generator=g), at)
                at += T
    for step in range(3):
        _step(paged, flat, g, [n + step if n else -1 for n in lens])
    _same_cache(paged, flat, [s for s, n in enumerate(lens) if n])


@pytest.mark.parametrize("captured", [False, True])
def test_fork_decode_release_compact(model, captured):
    """One prompt, three children next to it: every step over the shared
    prefix; the page the fork falls into is copied when written; a released
    child's pages are used again; a compaction in between changes nothing."""
    paged, flat = _stacks(model)
    g = torch.Generator(device=DEV).manual_seed(2)
    _prefill(paged, flat, 0, torch.randn(300, 2048, device=DEV, generator=g), 0)
    _prefill(paged, flat, 5, torch.randn(90, 2048, device=DEV, generator=g), 0)
    graph = None
    if captured:
        graph = {"x": torch.zeros(SLOTS, 2048, device=DEV), "pos": torch.full((SLOTS,), -1, dtype=torch.int32, device=DEV)}
        torch.cuda.synchronize()
        keep = [{k: t.clone() for k, t in S.items()} for S in paged.states]
        paged.decode_step(graph["x"], graph["pos"])   # (every slot idle: no page is touched)
        torch.cuda.synchronize()
        graph["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph["graph"]):
            paged.decode_step(graph["x"], graph["pos"])
        for S, K in zip(paged.states, keep):
            for k, t in S.items():
                t.copy_(K[k])
    used = int((paged.pages.refs > 0).sum())
    paged.fork(0, [1, 2, 3])
    _flat_fork(flat, 0, [1, 2, 3])
    assert int((paged.pages.refs > 0).sum()) == used
    assert paged.pages.group.tolist() == [0, 0, 0, 0, -1, -1]
    pos = [300, 300, 300, 300, -1, 90]
    for step in range(3):
        _step(paged, flat, g, [p + step if p >= 0 else -1 for p in pos], graph)
    assert int((paged.pages.refs > 0).sum()) == used + 3      # 300 falls inside a page: one each, the last holder keeps it
    assert paged.pages.shared_len.tolist()[:4] == [256] * 4
    _same_cache(paged, flat, [0, 1, 2, 3, 5])
    paged.release(1)
    moved = paged.compact()
    assert moved == used + 2
    _same_cache(paged, flat, [0, 2, 3, 5])
    paged.fork(2, [1])
    _flat_fork(flat, 2, [1])
    for step in range(3, 5):
        _step(paged, flat, g, [p + step if p >= 0 else -1 for p in pos], graph)
    _same_cache(paged, flat, [0, 1, 2, 3, 5])


@pytest.mark.parametrize("captured", [False, True])
def test_slots_that_sit_out_steps(model, captured):
    """A slot between two slices of its prompt and one between two steps sit out
    other slots' steps: they go on as if those had not been (the same kernels on
    the same inputs: the same bits as in a stack that has them alone, but for the
    split of the attention, 2e-5 of a step's largest update: 5e-6 for each of the two
    attention layers of either). A parked slot is forked; a sequence begins by a step."""
    paged, _ = _stacks(model)
    alone, _ = _stacks(model)
    g = torch.Generator(device=DEV).manual_seed(5)
    rows = lambda n: torch.randn(n, 2048, device=DEV, generator=g)
    graph = None
    if captured:
        graph = {"x": torch.zeros(SLOTS, 2048, device=DEV), "pos": torch.full((SLOTS,), -1, dtype=torch.int32, device=DEV)}
        paged.decode_step(graph["x"], graph["pos"])
        torch.cuda.synchronize()
        graph["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph["graph"]):
            paged.decode_step(graph["x"], graph["pos"])

    def steps(st, positions, xs, graph=None):
        st.reserve(positions)
        x, pos = xs.clone(), torch.tensor(positions, dtype=torch.int32, device=DEV)
        if graph is None:
            st.decode_step(x, pos)
            return x
        graph["x"].copy_(x)
        graph["pos"].copy_(pos)
        graph["graph"].replay()
        return graph["x"].clone()

    def close(a, b, x):
        assert not torch.isnan(a).any()
        assert float((a - b).abs().max() / (b - x).abs().max()) <= 2e-5

    first, second, other = rows(150), rows(140), rows(200)
    for st in (paged, alone):
        a, b = first.clone(), other.clone()
        st.prefill(0, a)
        st.prefill(3, b)
    # slot 3 steps while slot 0 waits for its second slice
    for i in range(3):
        xs = rows(SLOTS)
        got = steps(paged, [-1, -1, -1, 200 + i, -1, -1], xs, graph)
        want = steps(alone, [-1, -1, -1, 200 + i, -1, -1], xs)
        close(got[3], want[3], xs[3])
    a, b = second.clone(), second.clone()
    paged.prefill(0, a, 150)
    lone, _ = _stacks(model)
    c = first.clone()
    lone.prefill(0, c)
    lone.prefill(0, b, 150)
    assert torch.equal(a, b)
    with pytest.raises(ValueError):
        paged.prefill(0, second.clone(), 150)
    # slot 3 sits out, slot 0 steps; slot 3 is forked meanwhile; slot 5 begins by a step
    xs = rows(SLOTS)
    close(steps(paged, [290, -1, -1, -1, -1, -1], xs, graph)[0], steps(lone, [290, -1, -1, -1, -1, -1], xs)[0], xs[0])
    paged.fork(3, [4])
    alone.fork(3, [4])
    fresh, _ = _stacks(model)
    xs = rows(SLOTS)
    got = steps(paged, [-1, -1, -1, 203, 203, 0], xs, graph)
    want = steps(alone, [-1, -1, -1, 203, 203, -1], xs)
    for s in (3, 4):
        close(got[s], want[s], xs[s])
    close(got[5], steps(fresh, [-1] * 5 + [0], xs)[5], xs[5])


def test_calls_of_a_stack_without_pages(model):
    _, flat = _stacks(model)
    for call in (lambda: flat.reserve([-1] * SLOTS), lambda: flat.prefill(0, torch.zeros(4, 2048, device=DEV)),
                 lambda: flat.fork(0, [1]), lambda: flat.release(0), lambda: flat.compact()):
        with pytest.raises(ValueError):
            call()


def test_out_of_pages_changes_nothing(model):
    from qff.pages import OutOfPages
    paged, _ = _stacks(model, pages=3)
    x = torch.randn(200, 2048, device=DEV)
    keep = x.clone()
    with pytest.raises(OutOfPages):
        paged.prefill(0, x)
    assert torch.equal(x, keep) and paged.pages.free_pages == 3
    with pytest.raises(ValueError):
        paged.prefill(0, torch.zeros(513, 2048, device=DEV))    # more than the context's slice
    assert paged.pages.free_pages == 3


def test_out_of_pages_in_a_step_leaves_the_slots_before_whole(model):
    """Two children write into the page they share with their parent, one page
    is free: the first has its copy, the second is refused."""
    from qff.pages import OutOfPages
    paged, _ = _stacks(model, pages=2)
    paged.prefill(0, torch.randn(40, 2048, device=DEV))
    paged.fork(0, [1, 2])
    with pytest.raises(ValueError):
        paged.fork(0, [3, 1])
    assert paged.pages.lengths == [40, 40, 40, 0, 0, 0]
    with pytest.raises(OutOfPages):
        paged.reserve([-1, 40, 40, -1, -1, -1])
    first, copy = paged.pages.pages_of(0)[0], paged.pages.pages_of(1)[0]
    assert copy != first and paged.pages.pages_of(2) == [first]
    for kind, S in zip(paged.kinds, paged.states):
        if kind == "gqa":
            assert torch.equal(S["k_pages"][copy, :40], S["k_pages"][first, :40])
            assert torch.equal(S["v_pages"][copy, :40], S["v_pages"][first, :40])
