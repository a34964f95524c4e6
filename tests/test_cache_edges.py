"""Values, layouts, sizes and threads at which the operators on a KV cache can go wrong and that the tests of their ordinary
range do not reach.  Error bounds as in test_cache_ops.py."""
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from kuipy import _ffi
from oracle import kuiops_oracle as O
from test_cache_ops import DT, check_evict, check_mass, check_tree, f64, lens_t, tree_inputs


def test_error_codes_name_one_kernel():
    """The error word says which wait gave up: no two kernels share a code."""
    owner = {}
    for src in sorted((Path(_ffi.__file__).resolve().parents[1] / "csrc").glob("*.cu*")):
        for code in re.findall(r"atomic(?:CAS\(\s*(?:p\.)?err, 0u|Exch\((?:p\.)?err), (\d+)u", src.read_text()):
            assert owner.setdefault(int(code), src.name) == src.name, (code, owner[int(code)], src.name)
    assert len(set(owner.values())) >= 6


# ------------------------------------------------------------------------------------------------
# tree attention: infinities and NaN in visible values of the cache
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n,h,hk,l,s,d,lens,dtype,scale", [
    (2, 4, 2, 2, 200, 128, [200, 67], "bf16", None),             # 4 rows per KV head
    (1, 8, 2, 8, 130, 128, [129], "f16", None),                  # 32
    (2, 8, 2, 9, 130, 128, [130, 64], "bf16", None),             # 36
    (1, 8, 2, 16, 90, 64, [80], "f16", None),                    # 64
    (1, 8, 2, 17, 129, 128, [128], "bf16", None),                # 68
    (1, 8, 2, 32, 100, 64, [97], "f16", None),                   # 128
    (1, 4, 1, 70, 90, 128, [77], "bf16", None),                  # 280: three tiles of rows
    (1, 8, 2, 5, 5000, 128, [4999], "f16", None),                # keys split over CTAs, joined from records
    (1, 8, 2, 24, 5000, 128, [4999], "bf16", None),
    (40, 16, 8, 3, 200, 128, [71 + (i * 29) % 130 for i in range(40)], "bf16", None),      # CTAs that walk several units
    (2, 6, 3, 5, 77, 80, [70, 77], "f16", None),                 # head dims that are no multiple of 64
    (1, 4, 2, 6, 130, 40, [127], "bf16", None),
    (1, 8, 2, 32, 300, 128, [300], "f16", 0.5),                  # weights below fp16's least, whose values still count
    (1, 4, 2, 2, 300, 128, [300], "f16", 0.5),
    (1, 2, 2, 4, 99, 33, [90], "bf16", None),                    # SIMT kernel
    (1, 8, 2, 9, 1500, 64, [1400], "f32", None),
])
def test_tree_visible_values_that_are_not_finite(cuda, n, h, hk, l, s, d, lens, dtype, scale):
    """A cache value that overflowed reaches every row that sees it as in a sum with positive weights: an infinity, or NaN
    where both signs or a NaN meet; the other columns and the other heads stay as they are."""
    Q, K, V, Kd, Vd, mask = tree_inputs(n, h, hk, l, s, d, dtype, seed=l + s)
    inf, nan = float("inf"), float("nan")
    for b in {0, n - 1}:
        end = lens[b]
        V[b, 0, 0, 0], V[b, 0, end - 1, 1] = inf, -inf
        V[b, 0, 3, 2], V[b, 0, end // 2, 2] = inf, -inf
        V[b, 0, 5, 3], V[b, 0, 6, 4], V[b, 0, 7, 4] = nan, inf, inf
        V[b, hk - 1, end // 3, d - 1] = -inf
        Vd[b, 0, 0, 0], Vd[b, 0, l // 2, 1] = -inf, -inf                        # meets the cache's +inf; adds to its -inf
    out, lse = _ffi.sdpa_tree(Q, K, V, lens_t(lens), Kd, Vd, mask, scale=scale)
    check_tree(Q, K, V, lens, Kd, Vd, mask, dtype, out, lse, scale=scale)
    want = O.sdpa_tree(f64(Q), f64(K), f64(V), lens, f64(Kd), f64(Vd), mask.cpu().numpy(), scale)[0]
    odd = np.isinf(want)
    assert odd.any() and np.isnan(want).any() and np.array_equal(f64(out)[odd], want[odd])     # the sign too
    again, _ = _ffi.sdpa_tree(Q, K, V, lens_t(lens), Kd, Vd, mask, scale=scale)
    assert torch.equal(out.nan_to_num(5.0), again.nan_to_num(5.0)) and _ffi.tc_error() == 0


# ------------------------------------------------------------------------------------------------
# host threads
# ------------------------------------------------------------------------------------------------
class Recorder:
    """Makes the library's calls and keeps the arguments of the last one."""
    def __init__(self, real):
        self.real = real

    def __getattr__(self, name):
        def fn(*a):
            self.last = (name, a)
            return getattr(self.real, name)(*a)
        return fn


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["tree", "mass", "sdpa"])
def test_host_threads_with_different_head_sizes(cuda, op, monkeypatch):
    """One kernel serves heads of all sizes and takes more than the default shared memory for wide ones: calls of two sizes from two
    threads at once all launch, and give what they give alone."""
    from threading import Barrier, Thread

    def call(e, ev):
        g = torch.Generator(device="cuda").manual_seed(e)
        r = lambda *sh: torch.randn(*sh, generator=g, device="cuda")                             # noqa: E731
        if op == "tree":
            a = (r(1, 2, 8, e), r(1, 2, 32, e), r(1, 2, 32, ev), None, r(1, 2, 8, e), r(1, 2, 8, ev), torch.ones(8, 8, dtype=torch.bool, device="cuda"))
            return lambda: _ffi.sdpa_tree(*a)
        if op == "mass":
            a = (r(1, 2, 8, e), r(1, 2, 32, e), torch.full((1, 2, 8), 3.0, device="cuda"))
            return lambda: (_ffi.attn_mass(*a, is_causal=False),)
        a = (r(1, 2, 16, e), r(1, 2, 32, e), r(1, 2, 32, ev))
        return lambda: _ffi.sdpa(*a)

    real, rec = _ffi.lib(), Recorder(_ffi.lib())
    monkeypatch.setattr(_ffi, "lib", lambda: rec)
    made = []                                            # per thread: result, function and arguments, and what keeps them alive
    for e in (1024, 420, 1024, 420):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            fn = call(e, 256)
            made.append((fn(), rec.last, fn, stream))
    monkeypatch.undo()
    torch.cuda.synchronize()
    alone = [res[0].clone() for res, *_ in made]
    for res, *_ in made:
        res[0].fill_(7.0)
    torch.cuda.synchronize()
    codes, start = [set(), set(), set(), set()], Barrier(4)

    def work(i):
        name, args = made[i][1]
        fn = getattr(real, name)
        start.wait()
        for _ in range(5000):                            # nothing but the library's call: the threads meet inside it
            codes[i].add(fn(*args))
    threads = [Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [{_ffi.OK}] * 4
    assert all(torch.equal(a, res[0]) for a, (res, *_) in zip(alone, made))


@pytest.mark.gpu
def test_first_call_of_a_host_thread(cuda, monkeypatch):
    """A thread whose first use of the GPU is one of the library's calls."""
    from threading import Thread
    real, rec = _ffi.lib(), Recorder(_ffi.lib())
    Q, K, V, Kd, Vd, mask = tree_inputs(1, 8, 2, 5, 300, 128, "bf16", seed=3)
    A, B = torch.randn(64, 256, device="cuda").bfloat16(), torch.randn(128, 256, device="cuda").bfloat16()
    lse = torch.full((1, 8, 5), 4.0, device="cuda")
    monkeypatch.setattr(_ffi, "lib", lambda: rec)
    made = []
    for fn in (lambda: _ffi.gemm(A, B, trans_b=True), lambda: _ffi.sdpa(Q, K, V, is_causal=True), lambda: _ffi.sdpa(K, K, V, is_causal=True),
               lambda: _ffi.sdpa_tree(Q, K, V, None, Kd, Vd, mask), lambda: _ffi.attn_mass(Q, K, lse)):
        res = fn()
        made.append((res if isinstance(res, tuple) else (res,), rec.last))
    monkeypatch.undo()
    torch.cuda.synchronize()
    want = [res[0].clone() for res, _ in made]
    for res, _ in made:
        res[0].zero_()
    torch.cuda.synchronize()
    codes = []
    for _, (name, args) in made:
        t = Thread(target=lambda: codes.append(getattr(real, name)(*args)))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert codes == [_ffi.OK] * 5 and all(torch.equal(a, res[0]) for a, (res, _) in zip(want, made))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,l", [("bf16", 5), ("bf16", 24), ("f32", 5)])
def test_host_threads_on_one_stream(cuda, dtype, l, monkeypatch):
    """Calls that leave records for a joining kernel, from several threads into one stream: they share the stream's workspace, and
    each gets its own result."""
    from threading import Barrier, Thread
    real, rec = _ffi.lib(), Recorder(_ffi.lib())
    monkeypatch.setattr(_ffi, "lib", lambda: rec)
    made = []
    for seed in range(3):
        inputs = tree_inputs(1, 8, 2, l, 3000, 128, dtype, seed=seed)
        Q, K, V, Kd, Vd, mask = inputs
        made.append((_ffi.sdpa_tree(Q, K, V, None, Kd, Vd, mask), rec.last, inputs))
    monkeypatch.undo()
    torch.cuda.synchronize()
    alone = [[t.clone() for t in res] for res, *_ in made]
    start, wrong, codes = Barrier(3), [0, 0, 0], set()
    for _ in range(20):
        for res, *_ in made:
            res[0].fill_(7.0)
        torch.cuda.synchronize()

        def work(i):
            name, args = made[i][1]
            fn = getattr(real, name)
            start.wait()
            for _ in range(100):
                codes.add(fn(*args))
        threads = [Thread(target=work, args=(i,)) for i in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for i, (res, *_) in enumerate(made):
            wrong[i] += not all(torch.equal(a, b) for a, b in zip(alone[i], res))
    assert wrong == [0, 0, 0] and codes == {_ffi.OK}


# ------------------------------------------------------------------------------------------------
# layouts that are written to
# ------------------------------------------------------------------------------------------------
def test_rows_that_share_memory_are_not_written():
    """A cache or output whose (entry, head, row) steps coincide has rows on top of each other; dense ones in any order of dimensions,
    slices and gaps do not."""
    flat = torch.zeros(4096)
    view = lambda shape, stride: flat.as_strided(shape, stride)                                  # noqa: E731
    for shape, stride in (((2, 3, 5, 8), (120, 40, 8, 1)), ((2, 3, 5, 8), (120, 8, 24, 1)), ((2, 3, 5, 8), (8, 80, 16, 1)), ((2, 3, 5, 8), (400, 50, 9, 1)),
                          ((1, 3, 5, 8), (0, 40, 8, 1)), ((2, 1, 5, 8), (40, 0, 8, 1)), ((2, 3, 1, 8), (24, 8, 0, 1)), ((2, 3, 5, 1), (15, 5, 1, 7)),
                          ((1, 1, 1, 8), (0, 0, 0, 1))):
        assert _ffi._own_rows(view(shape, stride)), stride
    for shape, stride in (((2, 3, 5, 8), (8, 8, 8, 1)), ((2, 3, 5, 8), (120, 8, 8, 1)), ((2, 3, 5, 8), (40, 40, 8, 1)), ((2, 3, 5, 8), (120, 39, 8, 1)),
                          ((2, 3, 5, 8), (119, 40, 8, 1)), ((2, 3, 5, 8), (0, 40, 8, 1)), ((2, 3, 5, 8), (120, 40, 8, 2)), ((2, 3, 5, 8), (120, 40, 7, 1))):
        t = view(shape, stride)
        assert not _ffi._own_rows(t), stride
        with pytest.raises(_ffi.KuiopsError) as err:
            _ffi.kv_append(t, t, torch.zeros(2, dtype=torch.int64), t, t)
        assert "rows of their own" in str(err.value)


# ------------------------------------------------------------------------------------------------
# eviction whose moves take a launch of their own (more than 16 MiB could move)
# ------------------------------------------------------------------------------------------------
def evict_inputs(n, hk, cap, d, dv, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if dtype == "u8":
        r = lambda *s: torch.randint(0, 256, s, generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    else:
        r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(DT[dtype])                 # noqa: E731
    return r, torch.exp(2 * torch.randn(n, hk, cap, generator=g, device="cuda"))


def spreads(n, hk, cap, budget, d, dv, size):
    return n * hk * min(budget, cap - budget) * (d + dv) * size > 16 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("n,hk,cap,budget,d,dv,dtype,lens,sinks,recent", [
    (6, 8, 2500, 1001, 128, 128, "bf16", [2500, 900, 0], 4, 64),           # a budget of no whole chunks, several layers, rows within it
    (4, 8, 2200, 1056, 128, 128, "f16", [2200, 1056, 1057, 1 << 40], 0, 0),
    (2, 4, 9000, 4097, 128, 128, "bf16", [9000, 4098], 1, 4096),
    (16, 8, 700, 257, 128, 64, "f32", [700, 258, 600, 257], 0, 257),
    (4, 4, 30000, 14001, 33, 7, "bf16", [29999, 14002], 2, 100),           # 2-byte units
    (4, 2, 17000, 8191, 37, 35, "f32", [17000], 0, 8191),                  # 4-byte units
    (4, 2, 24000, 11003, 100, 101, "u8", [23000, 24000], 4, 10),           # single bytes
])
def test_evict_moves_in_a_launch_of_their_own(cuda, n, hk, cap, budget, d, dv, dtype, lens, sinks, recent):
    r, mass = evict_inputs(n, hk, cap, d, dv, dtype, budget)
    K, V = r(n, hk, cap, d), r(n, hk, cap, dv)
    assert spreads(n, hk, cap, budget, d, dv, K.element_size())
    check_evict(K, V, mass, lens, budget, sinks=sinks, recent=recent)


@pytest.mark.gpu
def test_evict_moves_in_a_launch_of_their_own_strides_and_positions(cuda):
    """Rows off the 16-byte grid, slices, (entry, slot, head) order, and positions out of order as earlier evictions leave them."""
    n, hk, cap, budget, d = 4, 4, 5000, 2177, 128
    r, mass = evict_inputs(n, hk, cap, d, d, "bf16", 1)
    assert spreads(n, hk, cap, budget, d, d, 2)
    pos = torch.stack([torch.randperm(9000, generator=torch.Generator().manual_seed(i))[:cap] for i in range(n * hk)]).view(n, hk, cap).int().cuda()
    V = r(n, cap, hk, d).transpose(1, 2)
    for K in (r(n, hk, cap + 9, d)[:, :, 9:], r(n * hk * cap * d + 1)[1:].view(n, hk, cap, d), r(n, hk, cap, d + 1)[..., 1:]):
        check_evict(K, V.clone(), mass, [5000, 3001], budget, pos=pos, next_pos=[9000, 9000], sinks=30, recent=500)


@pytest.mark.gpu
def test_evict_moves_in_a_launch_of_their_own_captured(cuda):
    n, hk, cap, budget, d = 5, 8, 2500, 1001, 128
    r, mass = evict_inputs(n, hk, cap, d, d, "bf16", 2)
    K0, V0 = r(n, hk, cap, d), r(n, hk, cap, d)
    assert spreads(n, hk, cap, budget, d, d, 2)
    K, V, lens = K0.clone(), V0.clone(), lens_t([2500])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = _ffi.kv_evict(K, V, mass, lens, budget, sinks=4, recent=64)
    for k, change in enumerate(([2500], [1001], [2111])):
        K.copy_(K0)
        V.copy_(V0)
        lens.copy_(lens_t(change))
        mass.copy_(mass.roll(k + 1, 2))
        graph.replay()
        torch.cuda.synchronize()
        K1, V1 = K0.clone(), V0.clone()
        want = _ffi.kv_evict(K1, V1, mass, lens, budget, sinks=4, recent=64)
        assert all(torch.equal(a, b) for a, b in zip(got + (K, V), want + (K1, V1)))
    del graph


@pytest.mark.gpu
def test_evict_offsets_beyond_32_bits(cuda):
    """The last entry's rows lie 2^31 elements behind the first one's."""
    n, hk, cap, budget, d, used = 3, 8, 1 << 20, 2003, 128, 2600
    K, V = (torch.empty(n, hk, cap, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    mass = torch.zeros(n, hk, cap, device="cuda")
    r, m = evict_inputs(1, hk, used, d, d, "bf16", 3)
    k, v = r(1, hk, used, d), r(1, hk, used, d)
    K[2:, :, :used], V[2:, :, :used], mass[2:, :, :used] = k, v, m
    assert spreads(n, hk, cap, budget, d, d, 2)
    lens, mass_out, pos, src = _ffi.kv_evict(K, V, mass, lens_t([0, 0, used]), budget, sinks=4, recent=100)
    want = _ffi.kv_evict(k, v, m, lens_t([used]), budget, sinks=4, recent=100)
    assert lens.tolist() == [0, 0, budget] and torch.equal(src[2:], want[3]) and bool((src[:2] == -1).all())
    assert torch.equal(K[2:, :, :used], k) and torch.equal(V[2:, :, :used], v)
    assert torch.equal(mass_out[2:, :, :used], want[1]) and torch.equal(pos[2:, :, :used], want[2])
    assert float(mass_out[:, :, used:].abs().max()) == 0.0 and bool((pos[:, :, used:] == -1).all())


# ------------------------------------------------------------------------------------------------
# attention mass with a limit per row, as a verified step asks for it
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("layers,g,h,hk,l,s,d,dtype", [
    (3, 2, 8, 2, 17, 300, 128, "bf16"),               # 68 rows a KV head: one tile of rows that streams
    (2, 3, 32, 8, 27, 700, 128, "f16"),               # 108
    (4, 1, 8, 2, 32, 129, 64, "bf16"),                # 128
    (2, 2, 8, 2, 33, 260, 128, "bf16"),               # two tiles
    (2, 3, 6, 2, 200, 150, 64, "f16"),                # five tiles, fewer keys than rows
    (1, 2, 7, 1, 64, 1000, 80, "bf16"),               # 448 rows under seven heads
    (32, 1, 32, 8, 27, 130, 128, "bf16"),             # every layer of a deep model
    (2, 2, 8, 2, 20, 200, 64, "f32"),
])
def test_attn_mass_row_limits_with_many_rows(cuda, layers, g, h, hk, l, s, d, dtype):
    """Most rows count for nothing (nodes that were not accepted), some for a few keys, some for more than there are; one sequence
    counts for none at all; entry b of the layers uses limits b % g."""
    n = layers * g
    gen = torch.Generator().manual_seed(l + s)
    qkv = torch.randn(n * l, (h + 2 * hk) * d, generator=gen).to(DT[dtype]).cuda()
    Q = qkv.as_strided((n, h, l, d), (l * qkv.shape[1], d, qkv.shape[1], 1))
    K = torch.randn(n, hk, s, d, generator=gen).to(DT[dtype]).cuda()
    lse = torch.randn(n, h, l, generator=gen).cuda() * 0.1 + float(np.log(s))
    lens = [s - (b * 31) % (s // 2) for b in range(g)]
    lim = [[0] * l for _ in range(g)]
    for b in range(g):
        for t, i in enumerate(sorted(torch.randperm(l, generator=gen)[:max(2, l // 8)].tolist())):
            lim[b][i] = lens[b] - 5 + t
        lim[b][0], lim[b][l - 1], lim[b][l // 2], lim[b][l // 3] = 1, 1 << 40, -3, 128
    if g > 2:
        lim[2] = [0] * l
    mass = torch.rand(n, hk, s, generator=gen).cuda()
    out = _ffi.attn_mass(Q, K, lse, kv_lens=lens_t(lens), q_lens=lens_t(lim), mass=mass)
    check_mass(Q, K, lse, lens * layers, lim * layers, mass, out)
    assert torch.equal(out[0, :, lens[0]:], mass[0, :, lens[0]:])
    if g > 2:
        assert torch.equal(out[2::g], mass[2::g])
    inplace = mass.clone()
    _ffi.attn_mass(Q, K, lse, kv_lens=lens_t(lens), q_lens=lens_t(lim), mass=inplace, out=inplace)
    assert torch.equal(inplace, out) and _ffi.tc_error() == 0
    # the limits alone say how many entries share them
    alone = _ffi.attn_mass(Q, K, lse, q_lens=lens_t(lim))
    check_mass(Q, K, lse, [s] * n, lim * layers, None, alone)
