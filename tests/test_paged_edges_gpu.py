"""Paged key-value cache on the GPU where values, arguments or calls are extreme: against definitions in 64 bits."""
import pytest
import torch

from _paged import attention_ref, make_cache, tokens_of

pytestmark = pytest.mark.gpu


def _F():
    from incin_b200.ops import functional as F
    return F


def _code():
    """The status word, cleared: 0, 6 for an index outside its tensors, 1 to 5 for a wait that ran out."""
    from incin_b200.ops import gemm as G
    word = G.status_word(torch.device("cuda", torch.cuda.current_device()))
    code = int(word.item())
    word.zero_()
    return code


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _reference(q, k, v, table, lengths, offsets, scale):
    """Softmax over the visible tokens in 64 bits and the weights' sum of |v|, ``[rows, heads, D]`` each."""
    hq, hkv = q.shape[1], k.shape[1]
    out, spread = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for s, n in enumerate(lengths.tolist()):
        a, b = int(offsets[s]), int(offsets[s + 1])
        kk, vv = (tokens_of(t, table, s, n).repeat_interleave(hq // hkv, 0) for t in (k, v))
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - (b - a), n, device="cuda")[:, None]
        p = torch.softmax((q[a:b].double().transpose(0, 1) @ kk.mT * scale).masked_fill(~seen, float("-inf")), -1)
        out[a:b], spread[a:b] = (p @ vv).transpose(0, 1), (p @ vv.abs()).transpose(0, 1)
    return out, spread


@pytest.mark.parametrize("scale,factor", [(1e4, 1), (1e8, 1), (1e10, 1), (1e12, 1), (1e30, 1), (1e38, 1), (None, 512)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,D", [(6, 2, 64), (24, 8, 128)])
def test_large_scales(scale, factor, dtype, hq, hkv, D):
    """Scores are whole numbers, so that 32 bits hold them exactly and other scores than the largest weigh exp(-1e4) or less: the
    rows are means over the largest scores' values.  Keys of one CTA, split keys, single tokens; a large scale, or large queries
    and keys."""
    g = torch.Generator().manual_seed(D)
    for new, past in (([200, 1, 3], [100, 0, 500]), ([70], [9000])):
        k, v, table, lens = make_cache([a + b for a, b in zip(new, past)], hkv, 32, D, dtype, "cuda", poison=False)
        k.copy_(torch.randint(-8, 9, k.shape, generator=g).to(dtype) * factor)
        q = torch.randint(-8, 9, (sum(new), hq, D), generator=g).to(dtype).cuda() * factor
        offsets = _i32(0, *torch.tensor(new).cumsum(0).tolist())
        ones = torch.arange(len(new) + 1)
        for x, offs, call in ((q, offsets, lambda: _F().prompt_attention(q, k, v, table, lens, offsets, scale=scale)),
                              (q[:len(new)], ones, lambda: _F().decode_attention(q[:len(new)], k, v, table, lens, scale=scale))):
            want, spread = _reference(x, k, v, table, lens, offs, D ** -0.5 if scale is None else scale)
            # equal weights of 1 (or a power of two), sums of a few values in 32 bits, one rounding
            bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -20 * spread + 2.0 ** -25
            got = call().double()
            assert _code() == 0
            assert ((got - want).abs() <= bound).all(), f"{(got.isnan()).sum().item()} NaN of {got.numel()}"


@pytest.mark.parametrize("kind", ["llama", "gpt2"])
def test_a_failed_step_is_taken_back(kind):
    """A step that raises half way leaves the cache as it was: the next one gives what it gives on a cache without the failure."""
    from incin_b200.cache import PagedCache
    from incin_b200.models.gpt2 import GPT2, GPT2Config
    from incin_b200.models.llama import Llama, LlamaConfig
    model = (Llama(LlamaConfig.tiny(), seed=1) if kind == "llama" else GPT2(GPT2Config.tiny(), seed=1)).cuda().to(torch.bfloat16)
    tok = torch.randint(0, 500, (80,), generator=torch.Generator().manual_seed(2)).cuda()
    outs = []
    for fail in (False, True):
        c = PagedCache.of(model, pages=20, page_size=16)
        a = c.new()
        model.extend(tok[:30], c, [a], [30])
        b = c.fork(a)
        if fail:
            block, real = model.blocks[1], model.blocks[1].extend
            block.extend = lambda *args: (real(*args), torch.empty(1 << 62))[0]       # out of memory behind the attention
            for tokens, counts in ((tok[30:70], [30, 10]), (tok[30:32], None)):
                with pytest.raises(RuntimeError):
                    model.extend(tokens, c, [a, b], counts)
            del block.extend
            assert c.length(a) == c.length(b) == 30
        outs.append(model.extend(tok[30:40], c, [a, b], [7, 3]))
        assert _code() == 0
    assert torch.equal(*outs)


@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("bits", [24.5, 25.5, 30.0])
@pytest.mark.parametrize("D", [64, 128])
def test_small_weights_in_fp16(place, bits, D):
    """One key outweighs every other by 2^bits; the sum of the others' weights is still right.  fp16 keeps a weight within 2^-25
    below 2^-14 and P is held as 2^7 at a row's reference, which is at most 2^8 off the largest score: 2^-32 a key is lost at
    most, 2^-11 of a weight above that range."""
    n, hkv, rows = 16384, 4, 64
    k, v, table, _ = make_cache([n], hkv, 64, D, torch.float16, "cuda", poison=False)
    k.zero_()
    v.fill_(1.0)
    at = {"first": 0, "middle": n // 2 + 5, "last": n - 1 - rows}[place]
    z = torch.tensor(bits * 0.6931471805599453, dtype=torch.float16)
    k[table[0, at // 64].long(), :, at % 64, 0] = z.cuda()
    v[table[0, at // 64].long(), :, at % 64] = 0.0
    weight = float(torch.exp(-z.double()))
    q = torch.zeros(rows, 2 * hkv, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0

    def check(out, seen):
        tail = (seen - 1) * weight
        want = tail / (1 + tail)
        # half a step of the result and of each weight, exponentials and sums of 32 bits, what is lost of each weight
        bound = want * (2 * 2.0 ** -11 + 2.0 ** -14) + seen * 2.0 ** -32
        assert _code() == 0
        err = (out.double().cpu() - want[:, None, None]).abs()
        assert (err <= bound[:, None, None]).all(), f"{err.max().item():.3e} of {want[-1].item():.3e}"

    lens = _i32(*[n] * rows)
    check(_F().decode_attention(q, k, v, table.expand(rows, -1), lens, scale=1.0), torch.full((rows,), float(n)))
    check(_F().prompt_attention(q, k, v, table, lens[:1], _i32(0, rows), scale=1.0), torch.arange(n - rows + 1, n + 1).double())


def test_forward_mode_is_refused():
    """A tangent would be lost: refused like an input that wants a gradient."""
    import torch.autograd.forward_ad as fw
    F = _F()
    k, v, table, lens = make_cache([20, 3], 2, 16, 64, torch.bfloat16, "cuda", poison=False)
    q, x = _randn(2, 4, 64, dtype=torch.bfloat16), _randn(2, 8 * 64, dtype=torch.bfloat16)
    want = F.decode_attention(q, k, v, table, lens)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        for call in (lambda: F.decode_attention(dual(q), k, v, table, lens), lambda: F.prompt_attention(q, k, dual(v), table, lens, _i32(0, 1, 2)),
                     lambda: F.kv_append(dual(x), k, v, table, lens, n_heads=4), lambda: F.copy_pages(dual(k)[None], _i32(0), _i32(1))):
            with pytest.raises(RuntimeError, match="no backward pass"):
                call()
        assert torch.equal(F.decode_attention(q, k, v, table, lens), want)
    with pytest.raises(RuntimeError, match="no backward pass"):
        torch.func.jvp(lambda t: F.decode_attention(t, k, v, table, lens), (q,), (q,))


def test_writes_in_place_are_seen_by_autograd():
    """A value saved for a backward pass, written by an append or a page copy before that pass runs, is an error there."""
    F = _F()
    k, v, table, lens = make_cache([20, 3], 2, 16, 64, torch.bfloat16, "cuda", poison=False)
    x = _randn(2, 8 * 64, dtype=torch.bfloat16)
    for t, write in ((k, lambda: F.kv_append(x, k, v, table, lens, n_heads=4)), (v, lambda: F.kv_append(x, k, v, table, lens, n_heads=4)),
                     (k, lambda: F.copy_pages(k[None], _i32(0), _i32(1)))):
        w = torch.ones_like(t, requires_grad=True)
        loss = (w * t).sum()
        write()
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
    with torch.inference_mode():
        held = torch.zeros_like(k)
    F.kv_append(x, held, held.clone(), table, lens, n_heads=4)       # tensors without a counter are written all the same
    F.copy_pages(held[None], _i32(0), _i32(1))
    assert _code() == 0


def _pages(n=8):
    return torch.arange(n, device="cuda", dtype=torch.float32).view(n, 1, 1, 1).expand(n, 1, 4, 4).contiguous()


def test_copy_pages_own_copy_is_a_source_too():
    """A page that is its own copy may be others' source, as on the CPU."""
    for src, dst in (((0, 0), (0, 1)), ((0, 0, 3), (1, 0, 2)), ((4, 4, 4), (4, 5, 6))):
        st, cpu = _pages(), _pages().cpu()
        _F().copy_pages(st, _i32(*src), _i32(*dst))
        assert _code() == 0
        assert torch.equal(st.cpu(), _F().copy_pages(cpu, torch.tensor(src, dtype=torch.int32), torch.tensor(dst, dtype=torch.int32)))
    for src, dst, kept in (((3, 5), (5, 5), [5]), ((5, 3), (5, 5), [5])):      # ... but not a destination, on neither
        st = _pages()
        _F().copy_pages(st, _i32(*src), _i32(*dst))
        assert _code() == 6 and torch.equal(st, _pages())
        with pytest.raises(IndexError):
            _F().copy_pages(_pages().cpu(), torch.tensor(src, dtype=torch.int32), torch.tensor(dst, dtype=torch.int32))


def test_copy_pages_pairs_that_name_no_page_exclude_no_other():
    for src, dst, want in (((-1, 2), (5, 5), [0, 1, 2, 3, 4, 2, 6, 7]), ((2, 8, 3), (5, 5, 5), [0, 1, 2, 3, 4, 2, 6, 7]),
                           ((5, 3), (8, 5), [0, 1, 2, 3, 4, 3, 6, 7]), ((5, 3, 1), (-2, 5, 5), [0, 1, 2, 3, 4, 3, 6, 7])):
        st = _pages()
        _F().copy_pages(st, _i32(*src), _i32(*dst))
        assert _code() == 6 and st[:, 0, 0, 0].tolist() == want


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("D", [64, 128])
def test_non_finite_values_of_small_weight(bad, D):
    """A non-finite value that every row sees makes its element non-finite, however small its weight and wherever the keys are
    split: 0 times it is no number either."""
    new, past, hq, hkv = [40], [9000], 6, 2
    k, v, table, lens = make_cache([9040], hkv, 64, D, torch.bfloat16, "cuda", poison=False)
    q = torch.zeros(40, hq, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    k.zero_()
    for at in (5, 4000, 8000):
        kk, vv = k.clone(), v.clone()
        kk[table[0, 8990 // 64].long(), :, 8990 % 64, 0] = 1000.0       # outweighs all others by e^1000
        vv[table[0, at // 64].long(), 0, at % 64, 3] = bad
        for out in (_F().prompt_attention(q, kk, vv, table, lens, _i32(0, 40), scale=1.0), _F().decode_attention(q[:1], kk, vv, table, lens, scale=1.0)):
            odd = ~torch.isfinite(out)
            assert odd[:, :3, 3].all() and not odd[:, 3:].any() and odd.sum() == 3 * out.shape[0]
    assert _code() == 0


@pytest.mark.parametrize("seqs", [3, 70])
def test_offsets_outside_the_rows_are_reported(seqs):
    """Offsets that fall, are negative or pass the rows: reported by both operators that read them, wherever in a batch."""
    F = _F()
    hq, hkv, D, rows = 4, 2, 64, 30
    k, v, table, lens = make_cache([70] * seqs, hkv, 16, D, torch.bfloat16, "cuda", poison=False)
    q, x = _randn(rows, hq, D, dtype=torch.bfloat16), _randn(rows, (hq + 2 * hkv) * D, dtype=torch.bfloat16)
    cuts = sorted(min(i, rows) for i in range(seqs + 1))
    for at, value, code in ((0, 0, 0), (seqs, rows, 0), (seqs, rows + 1, 6), (seqs, 2 ** 31 - 1, 6), (0, -1, 6), (0, -2 ** 31, 6), (seqs, 0, 6),
                            (1, rows + 5, 6), (seqs - 1, -7, 6)):
        offs = list(cuts)
        offs[at] = value
        good = all(0 <= a <= b <= rows for a, b in zip(offs, offs[1:]))
        assert good == (code == 0)
        F.prompt_attention(q, k, v, table, lens, _i32(*offs))
        assert _code() == code, f"prompt_attention: offsets[{at}] = {value}"
        F.kv_append(x, k.clone(), v.clone(), table, lens, _i32(*offs), n_heads=hq)
        assert _code() == code, f"kv_append: offsets[{at}] = {value}"


def test_a_cache_without_kernels_is_refused_at_once():
    """A model whose type has no kernels on CUDA is refused when its cache is made, not by the first call."""
    from incin_b200 import _native as nat
    from incin_b200.cache import PagedCache
    from incin_b200.models.llama import Llama, LlamaConfig
    with pytest.raises(nat.NativeError, match="float32"):
        PagedCache.of(Llama(LlamaConfig.tiny()).cuda(), pages=4)
    PagedCache.of(Llama(LlamaConfig.tiny()).cuda().half(), pages=4)
    PagedCache.of(Llama(LlamaConfig.tiny()), pages=4)


def test_no_wait_runs_out_for_odd_offsets():
    """Offsets that fall, start late, pass the rows or overlap: the status word tells of them, never of a wait; rows of one
    sequence alone are those of that run."""
    F = _F()
    hq, hkv, D, lengths = 4, 2, 64, [40, 50, 33]
    k, v, table, lens = make_cache(lengths, hkv, 16, D, torch.bfloat16, "cuda", poison=False)
    q = _randn(30, hq, D, dtype=torch.bfloat16)
    # offsets, whether they are in order, (sequence, first row, end, rows of it that no other sequence has)
    for offs, code, runs in (((5, 10, 20, 30), 0, [(0, 5, 10, range(5, 10)), (1, 10, 20, range(10, 20)), (2, 20, 30, range(20, 30))]),
                             ((0, 10, 10, 500), 6, [(0, 0, 10, range(10))]), ((0, 25, 10, 30), 6, [(0, 0, 25, range(10)), (2, 10, 30, range(25, 30))]),
                             ((-7, 3, 2 ** 31 - 1, 4), 6, []), ((30, 20, 10, 0), 6, []), ((0, 0, 0, 0), 0, [])):
        for _ in range(3):
            out = F.prompt_attention(q, k, v, table, lens, _i32(*offs))
        assert _code() == code
        for s, a, b, alone in runs:
            want, bound = attention_ref(q[a:b], k, v, table[s:s + 1], lens[s:s + 1], _i32(0, b - a), D ** -0.5)
            rows = torch.tensor(list(alone), device="cuda")
            assert ((out[rows].double() - want[rows - a]).abs() <= bound[rows - a]).all()


def test_no_wait_runs_out_for_idle_slots():
    """A captured batch whose slots empty and fill: idle ones have a row each by the prompt's offsets, more rows than tokens,
    which is reported as such and as nothing else."""
    F = _F()
    hq, hkv, D, S = 8, 2, 64, 5
    k, v, table, lens = make_cache([600] * S, hkv, 16, D, torch.bfloat16, "cuda", poison=False)
    q, offs = _randn(S, hq, D, dtype=torch.bfloat16), torch.arange(S + 1, dtype=torch.int32, device="cuda")
    F.prompt_attention(q, k, v, table, lens, offs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one, many = F.decode_attention(q, k, v, table, lens), F.prompt_attention(q, k, v, table, lens, offs)
    for now in ([600, 1, 17, 300, 2], [0, 1, 600, 0, 0], [0] * 5, [5, 0, 0, 0, 600], [1] * 5):
        lens.copy_(_i32(*now))
        for _ in range(3):
            graph.replay()
        assert _code() == (6 if 0 in now else 0)
        want, bound = attention_ref(q, k, v, table, lens, None, D ** -0.5)      # zeros for idle slots
        for out in (one, many):
            assert ((out.double() - want).abs() <= bound).all()
