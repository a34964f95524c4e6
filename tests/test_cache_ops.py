"""The operators on a KV cache across decode steps (sdpa_tree, tree_accept, kv_append, attn_mass, kv_evict) against
their definitions in 64 bits, at the sizes, masks, layouts and values where they can go wrong, and their refusals.

Error bounds (``u`` = half a step of the element type, 2^-8 for bf16, 2^-11 for fp16; fp32 arithmetic inside):
a score is a sum of e products, off by at most ds = (e + 8) 2^-24 scale sum|q k|; a weight exp(score - max) is then
off by a factor of at most 1 +- (2 ds + 2^-20 + keys 2^-24) (score and maximum, the exponential and the scaling to the
log2 domain of values below 32, the sum), and 16-bit types round each weight once more (u) before the product with
V; the result is rounded once (u)."""
import re
import struct
from pathlib import Path

import numpy as np
import pytest
import torch

from kuipy import _ffi
from oracle import kuiops_oracle as O

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 0.0}
HEADER = (Path(__file__).resolve().parent.parent / "include" / "kuiops.h").read_text()
P = 0x1000                               # a non-null pointer that is never dereferenced


def f64(t):
    return t.detach().double().cpu().numpy()


def tree_parents(n, l, g):
    """Random parents: node i hangs below one of the nodes before it."""
    par = torch.stack([torch.tensor([-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, l)]) for _ in range(n)])
    return par.long()


def ancestors(par):
    n, l = par.shape
    m = torch.zeros(n, l, l, dtype=torch.bool)
    for b in range(n):
        for i in range(l):
            j = i
            while j >= 0:
                m[b, i, j] = True
                j = int(par[b, j])
    return m


# ------------------------------------------------------------------------------------------------
# refusals (on the host; nothing is launched)
# ------------------------------------------------------------------------------------------------
def refused(fn, *a, **kw):
    with pytest.raises(_ffi.KuiopsError) as e:
        fn(*a, **kw)
    return e.value.code


def test_tree_refusals_of_the_binding():
    t = torch.zeros
    ok = dict(Q=t(2, 4, 3, 8), K=t(2, 2, 5, 8), V=t(2, 2, 5, 8), kv_lens=t(2, dtype=torch.int64), Kd=t(2, 2, 3, 8), Vd=t(2, 2, 3, 8),
              mask=t(3, 3, dtype=torch.bool))

    def call(**kw):
        a = {**ok, **kw}
        return refused(_ffi.sdpa_tree, a["Q"], a["K"], a["V"], a["kv_lens"], a["Kd"], a["Vd"], a["mask"], out=a.get("out"))
    for bad in (dict(Q=t(4, 3, 8)), dict(K=t(2, 2, 5, 16)), dict(V=t(2, 3, 5, 8)), dict(Kd=t(2, 2, 4, 8)), dict(Vd=t(1, 2, 3, 8)),
                dict(K=t(2, 2, 5, 8, dtype=torch.float16)), dict(mask=t(3, 4, dtype=torch.bool)), dict(mask=t(3, 3)),
                dict(mask=t(3, 3, 3, dtype=torch.bool)), dict(kv_lens=t(3, dtype=torch.int64)), dict(kv_lens=t(2, dtype=torch.int32)),
                dict(out=t(2, 4, 3, 9)), dict()):                     # the last: CPU tensors
        assert call(**bad) == _ffi.EINVAL, bad


def test_append_accept_mass_evict_refusals_of_the_binding():
    t, i64, i32 = torch.zeros, torch.int64, torch.int32
    ids = t(2, 5, dtype=i64)
    for a in ((t(5, dtype=i64), ids, t(2, 4, dtype=i64)), (t(4, dtype=i64), ids, ids), (t(5, dtype=i32), ids, ids),
              (t(5, dtype=i64), ids.float(), ids), (t(5, dtype=i64), ids, ids)):
        assert refused(_ffi.tree_accept, *a) == _ffi.EINVAL
    K, V, n1 = t(4, 2, 6, 8), t(4, 2, 6, 8), t(4, 2, 3, 8)
    lens = t(2, dtype=i64)
    for a, kw in (((K, V, t(3, dtype=i64), n1, n1), {}), ((K, t(4, 2, 7, 8), lens, n1, n1), {}), ((K, V, lens, n1, t(4, 2, 3, 9)), {}),
                  ((K, V, lens, n1.half(), n1), {}), ((K, V, lens, n1, n1), dict(path=t(2, 4, dtype=i64))),
                  ((K, V, lens, n1, n1), dict(counts=t(3, dtype=i64))), ((K, V, lens, n1, n1), dict(pos=t(4, 2, 6, dtype=i32))),
                  ((K, V, lens, n1, n1), dict(mass=t(4, 2, 5))), ((K.transpose(2, 3).contiguous().transpose(2, 3), V, lens, n1, n1), {}),
                  ((t(1, 2, 6, 8).expand(4, 2, 6, 8), V, lens, n1, n1), {}), ((K, V, lens, n1, n1), {})):
        assert refused(_ffi.kv_append, *a, **kw) == _ffi.EINVAL
    Q, lse, mass = t(4, 4, 3, 8), t(4, 4, 3), t(4, 2, 6)
    for a, kw in (((Q, t(4, 3, 6, 8), lse), {}), ((Q, K, t(4, 4, 2)), {}), ((Q, K, lse.double()), {}), ((Q, K, lse), dict(kv_lens=t(3, dtype=i64))),
                  ((Q, K, lse), dict(q_lens=t(2, 4, dtype=i64))), ((Q, K, lse), dict(mass=t(4, 2, 5))), ((Q, K, lse), dict(out=t(4, 2, 6).half())),
                  ((Q, K, lse), {})):
        assert refused(_ffi.attn_mass, *a, **kw) == _ffi.EINVAL
    for a, kw in (((K, V, mass, lens, 0), {}), ((K, V, mass, lens, 7), {}), ((K, V, mass, lens, 4), dict(sinks=3, recent=2)),
                  ((K, V, mass, lens, 4), dict(sinks=-1)), ((K, V, t(4, 2, 5), lens, 4), {}), ((K, V, mass, t(3, dtype=i64), 4), {}),
                  ((K, V, mass, lens, 4), dict(pos=t(4, 2, 6, dtype=i64))), ((K, V.half(), mass, lens, 4), {}), ((K, V, mass, lens, 4), {})):
        assert refused(_ffi.kv_evict, *a, **kw) == _ffi.EINVAL


def block(name):
    """Field names of an argument block of the header, in order, and a packer that takes them by name (0 unless given)."""
    body = re.search(r"typedef struct kuiops_%s_args \{(.*?)\}" % name, HEADER, re.S).group(1)
    fields = []
    for decl in body.split(";")[:-1]:
        kind = "q" if "*" in decl or "int64_t" in decl else ("f" if "float" in decl else "i" if re.search(r"\bint32_t", decl) else "I")
        names = re.sub(r"\b(const|void|float|u?int\d+_t)\b|\*", " ", decl)
        fields += [(x.strip(), "Q" if kind == "q" and "uint64" not in decl else kind.upper() if "uint64" in decl else kind) for x in names.split(",")]
    packer = getattr(_ffi, {"sdpa_tree": "_TREE_ARGS", "tree_accept": "_ACCEPT_ARGS", "kv_append": "_APPEND_ARGS", "attn_mass": "_MASS_ARGS", "kv_evict": "_EVICT_ARGS"}[name])
    fmt = packer.format if isinstance(packer.format, str) else packer.format.decode()
    assert struct.Struct("=" + "".join(k for _, k in fields)).size == packer.size == struct.calcsize("@" + fmt[1:])
    return [f for f, _ in fields], packer


def c_call(name, defaults):
    fields, packer = block(name)
    fn = getattr(_ffi.lib(), "kuiops_" + name)

    def call(**kw):
        a = {**defaults, **kw}
        assert set(a) <= set(fields), set(a) - set(fields)
        return fn(packer.pack(*[a.get(f, 0) for f in fields]), None)
    return call


def test_contracts_of_the_c_entries():
    L = _ffi.lib()
    for name in ("sdpa_tree", "tree_accept", "kv_append", "attn_mass", "kv_evict"):
        assert getattr(L, "kuiops_" + name)(None, None) == _ffi.EINVAL
    tree = c_call("sdpa_tree", dict(dtype=_ffi.BF16, n=1, h=4, h_kv=2, l=3, s=10, e=128, ev=128, q_sn=8, q_sh=128, k_sn=8, k_sh=128, v_sn=8, v_sh=128, dk_sh=128, dv_sh=128,
                                    o_sh=128, Q=P, K=P, V=P, DK=P, DV=P, mask=P, out=P, workspace=P,
                                    workspace_bytes=1 << 30, q_sl=128, k_ss=128, v_ss=128, dk_sl=128, dv_sl=128, o_sl=128, scale=0.1))
    assert tree(dtype=7) == tree(n=0) == tree(l=0) == tree(h=3) == tree(Q=0) == tree(K=0) == tree(mask=0) == tree(out=0) == _ffi.EINVAL
    assert tree(k_ss=64) == tree(mask_sk=(1 << 64) - 1) == tree(scale=float("nan")) == tree(scale=float("inf")) == _ffi.EINVAL
    assert tree(e=2048) == tree(ev=512) == _ffi.EUNSUPPORTED and tree(l=5000) == _ffi.ELIMIT
    need = L.kuiops_sdpa_tree_workspace_bytes(_ffi.BF16, 1, 4, 2, 3, 100000, 128, 128)
    assert need > 0
    assert tree(s=100000, workspace=0) == tree(s=100000, workspace_bytes=16) == tree(s=100000, workspace=P + 4) == _ffi.EWORKSPACE
    acc = c_call("tree_accept", dict(n=2, l=5, parents=P, draft=P, target=P, path=P, counts=P, next=P))
    assert acc(n=0) == acc(l=0) == acc(parents=0) == acc(next=0) == acc(parents_sn=4) == _ffi.EINVAL and acc(l=5000) == _ffi.ELIMIT
    app = c_call("kv_append", dict(elem_bytes=2, n=4, h_kv=2, l=3, cap=8, e=128, ev=128, lens_n=2, DK=P, DV=P, K=P, V=P, kv_lens=P,
                                   dk_sl=128, dv_sl=128, k_ss=128, v_ss=128))
    assert app(elem_bytes=8) == app(n=0) == app(cap=0) == app(kv_lens=0) == app(lens_n=3) == app(lens_n=0) == app(pos=P) == app(k_ss=64) == _ffi.EINVAL
    assert app(cap=0x7fffffff) == _ffi.ELIMIT
    mass = c_call("attn_mass", dict(dtype=_ffi.BF16, n=4, h=4, h_kv=2, l=3, s=8, e=128, lens_n=1, Q=P, K=P, lse=P, out=P, q_sl=128, k_ss=128, scale=0.1))
    assert mass(dtype=9) == mass(s=0) == mass(Q=0) == mass(lse=0) == mass(kv_lens=P, lens_n=3) == mass(scale=float("nan")) == _ffi.EINVAL
    assert mass(e=2000, q_sl=2000, k_ss=2000) == _ffi.EUNSUPPORTED
    evict = c_call("kv_evict", dict(elem_bytes=2, n=4, h_kv=2, cap=100, e=128, ev=128, lens_n=2, budget=10, K=P, V=P, mass=P, mass_out=P + 64, pos_out=P,
                                    src=P, kv_lens=P, lens_out=P + 8, k_ss=128, v_ss=128))
    assert evict(elem_bytes=3) == evict(budget=0) == evict(budget=101) == evict(sinks=6, recent=5) == evict(lens_n=3) == _ffi.EINVAL
    assert evict(sinks=0xFFFFFFFF, recent=2) == evict(mass=0) == evict(mass_out=P) == evict(lens_out=P) == _ffi.EINVAL


# ------------------------------------------------------------------------------------------------
# tree attention
# ------------------------------------------------------------------------------------------------
def tree_inputs(n, h, hk, l, s, d, dtype, seed, dv=None, masks="tree"):
    g = torch.Generator().manual_seed(seed)
    dt, dv = DT[dtype], dv or d
    r = lambda *sh: torch.randn(*sh, generator=g).to(dt).cuda()                                 # noqa: E731
    if masks == "tree":
        mask = ancestors(tree_parents(n, l, g))
    else:
        mask = torch.rand(n, l, l, generator=g) < 0.4
        mask[:, l // 2] = False                                  # a row that sees no drafted key
    return r(n, h, l, d), r(n, hk, s, d), r(n, hk, s, dv), r(n, hk, l, d), r(n, hk, l, dv), mask.cuda()


def check_tree(Q, K, V, lens, Kd, Vd, mask, dtype, out, lse, scale=None):
    m3 = mask if mask.dim() == 3 else mask[None]
    ll = lens if lens is not None else [K.shape[2]] * Q.shape[0]
    ro, rl, mag, reach = O.sdpa_tree(f64(Q), f64(K), f64(V), ll, f64(Kd), f64(Vd), m3.cpu().numpy(), scale)
    keys = K.shape[2] + Q.shape[2]
    ds = (Q.shape[3] + 8) * 2.0 ** -24 * reach
    wt = 2 * ds + 2.0 ** -20 + keys * 2.0 ** -24
    o, l_ = f64(out), f64(lse)
    assert np.array_equal(np.isnan(o), np.isnan(ro)) and np.array_equal(np.isinf(o), np.isinf(ro))
    assert np.array_equal(np.isneginf(l_), np.isneginf(rl))
    fin = np.isfinite(ro)
    tol = (wt + U[dtype]) * mag + (U[dtype] + 2.0 ** -22) * np.abs(ro) + 2.0 ** -24
    assert (np.abs(o - ro)[fin] <= tol[fin]).all(), (np.abs(o - ro)[fin] / tol[fin]).max()
    fin = np.isfinite(rl)
    tol = ds + 2.0 ** -20 + keys * 2.0 ** -24 + 2.0 ** -23 * np.abs(rl)
    assert (np.abs(l_ - rl)[fin] <= tol[fin]).all(), (np.abs(l_ - rl)[fin] / tol[fin]).max()


def lens_t(lens):
    return torch.tensor(lens, dtype=torch.int64).cuda()


TREE_CASES = [
    # n, h, hk, l, s, d, lens, dtype
    (1, 4, 4, 1, 64, 128, [64], "bf16"),                # one row, one tile exactly
    (2, 4, 2, 3, 70, 128, [65, 0], "bf16"),             # one key in the second tile; an empty cache
    (3, 8, 2, 8, 200, 128, [63, 1, 200], "f16"),        # 32 rows per KV head
    (2, 8, 2, 9, 130, 128, [130, 64], "bf16"),          # 36 rows
    (1, 8, 2, 16, 129, 128, [129], "f16"),              # 64 rows
    (1, 8, 2, 17, 129, 128, [128], "bf16"),             # 68 rows
    (1, 8, 2, 32, 100, 128, [97], "bf16"),              # 128 rows
    (2, 14, 2, 27, 66, 128, [66, 40], "bf16"),          # 7 heads per KV head, 189 rows
    (1, 4, 1, 70, 90, 128, [77], "f16"),                # two tiles of drafted keys
    (1, 3, 1, 130, 10, 128, [10], "bf16"),              # more drafted rows than a tile of rows, three heads
    (1, 8, 2, 5, 5000, 128, [4999], "bf16"),            # split over CTAs
    (2, 4, 2, 33, 3000, 128, [2990, 5], "f16"),         # split, ragged
    (2, 4, 2, 7, 150, 64, [150, 99], "bf16"),
    (1, 8, 1, 20, 2100, 64, [2049], "f16"),
    (2, 6, 3, 5, 77, 80, [70, 77], "bf16"),             # head dims that are no multiple of 64
    (1, 4, 2, 6, 130, 40, [127], "f16"),
    (1, 4, 2, 6, 130, 96, [128], "bf16"),
    (1, 2, 1, 5, 90, 72, [81], "f16"),
    (1, 2, 2, 4, 67, 33, [66], "bf16"),                 # odd head dim
    (1, 4, 2, 5, 600, 256, [513], "bf16"),
    (2, 4, 2, 6, 130, 128, [127, 31], "f32"),
    (1, 8, 2, 9, 1500, 64, [1400], "f32"),
    (1, 2, 2, 5, 40, 24, [0], "f32"),
    (1, 160, 1, 2, 70, 128, [65], "bf16"),              # more heads per KV head than a tile has rows
    # more units than CTAs: a CTA walks several, ends in the middle of one and goes on in the middle of another
    (80, 8, 8, 2, 260, 128, [(i * 37) % 261 for i in range(80)], "bf16"),
    (60, 16, 8, 12, 130, 64, [(i * 53) % 131 for i in range(60)], "f16"),
    (40, 16, 8, 24, 200, 128, [(i * 29) % 201 for i in range(40)], "bf16"),
    (24, 64, 8, 12, 300, 128, [300 - (i * 41) % 299 for i in range(24)], "bf16"),
    (18, 16, 2, 33, 700, 128, [(i * 97) % 701 for i in range(18)], "f16"),     # three tiles of rows
    (300, 2, 1, 1, 70, 128, [i % 71 for i in range(300)], "bf16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("masks", ["tree", "random"])
@pytest.mark.parametrize("case", TREE_CASES, ids=lambda c: "-".join(str(x) for x in c[:6] + c[7:] + (c[6][:3],)).replace(" ", ""))
def test_tree_attention(cuda, case, masks):
    n, h, hk, l, s, d, lens, dtype = case
    Q, K, V, Kd, Vd, mask = tree_inputs(n, h, hk, l, s, d, dtype, seed=l * 1000 + s + d, masks=masks)
    out, lse = _ffi.sdpa_tree(Q, K, V, lens_t(lens), Kd, Vd, mask)
    check_tree(Q, K, V, lens, Kd, Vd, mask, dtype, out, lse)
    again, lse2 = _ffi.sdpa_tree(Q, K, V, lens_t(lens), Kd, Vd, mask)
    assert torch.equal(out, again) and torch.equal(lse, lse2)          # no sum depends on timing
    assert _ffi.tc_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tree_masked_places_hold_anything(cuda, dtype):
    """Keys no row sees (cache slots behind the count, drafted rows masked for all) hold NaN and infinities; a drafted row
    that overflowed spoils the rows that see it, and no other."""
    n, h, hk, l, s, d = 2, 8, 2, 12, 150, 128
    Q, K, V, Kd, Vd, mask = tree_inputs(n, h, hk, l, s, d, dtype, seed=5)
    lens = [100, 0]
    for b in range(n):
        K[b, :, lens[b]:], V[b, :, lens[b]:] = float("nan"), float("inf")
    mask[:, :, 7] = False
    mask[:, 7, :] = False                                              # row 7 sees only the cache: nothing in entry 1
    Kd[:, :, 7], Vd[:, :, 7] = float("inf"), float("nan")
    Vd[0, 0, 3, 5] = float("inf")                                      # seen by 3 and its descendants
    Vd[0, 1, 4, 127] = float("nan")
    out, lse = _ffi.sdpa_tree(Q, K, V, lens_t(lens), Kd, Vd, mask)
    check_tree(Q, K, V, lens, Kd, Vd, mask, dtype, out, lse)
    assert (out[1, :, 7] == 0).all() and torch.isneginf(lse[1, :, 7]).all()
    assert bool(torch.isinf(out[0, 0, 3, 5])) and bool(torch.isnan(out[0, 4, 4, 127]))
    # a query row that is NaN spoils itself alone
    Q[0, 2, 1, 0] = float("nan")
    out, lse = _ffi.sdpa_tree(Q, K, V, lens_t(lens), Kd, Vd, mask)
    assert torch.isnan(out[0, 2, 1]).all() and torch.isnan(lse[0, 2, 1]) and torch.isfinite(out[0, 2, 2]).all()


@pytest.mark.gpu
def test_tree_large_scores_and_negative_scale(cuda):
    Q, K, V, Kd, Vd, mask = tree_inputs(1, 4, 2, 6, 300, 128, "bf16", seed=9)
    for scale in (1.0, 4.0, -0.2):                                     # steep softmax: the running maximum moves
        out, lse = _ffi.sdpa_tree(Q, K, V, lens_t([290]), Kd, Vd, mask, scale=scale)
        check_tree(Q, K, V, [290], Kd, Vd, mask, "bf16", out, lse, scale=scale)
    out, lse = _ffi.sdpa_tree(Q, K, V, lens_t([290]), Kd, Vd, mask, scale=0.0)     # the mean of what is seen
    check_tree(Q, K, V, [290], Kd, Vd, mask, "bf16", out, lse, scale=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f32", 64), ("bf16", 33)])
def test_tree_views_strides_and_shared_mask(cuda, dtype, d):
    """Rows inside packed projections, a sliced cache, a transposed output, one mask for all, no key counts, counts beyond
    the cache, no lse; and operands that start off a 16-byte boundary."""
    n, h, hk, l, s = 2, 4, 2, 11, 90
    g = torch.Generator().manual_seed(3)
    w = (h + 2 * hk) * d
    qkv = torch.randn(n * l, w + 8, generator=g).to(DT[dtype]).cuda()
    W = w + 8
    Q = qkv.as_strided((n, h, l, d), (l * W, d, W, 1))
    Kd, Vd = qkv.as_strided((n, hk, l, d), (l * W, d, W, 1), h * d), qkv.as_strided((n, hk, l, d), (l * W, d, W, 1), (h + hk) * d)
    cache = torch.randn(2, n, hk, s + 14, d, generator=g).to(DT[dtype]).cuda()
    K, V = cache[0][:, :, 3:3 + s], cache[1][:, :, 5:5 + s]
    mask = ancestors(tree_parents(1, l, g))[0].cuda()
    buf = torch.zeros(n, l, h, d, dtype=DT[dtype], device="cuda")
    out, lse = _ffi.sdpa_tree(Q, K, V, None, Kd, Vd, mask, out=buf.transpose(1, 2))
    check_tree(Q, K, V, None, Kd, Vd, mask, dtype, out, lse)
    assert out.data_ptr() == buf.data_ptr()
    for odd in (mask.t().contiguous().t(), torch.stack([mask] * 3, -1)[..., 1], mask.expand(n, l, l), mask[None]):       # the same mask, other strides
        again, _ = _ffi.sdpa_tree(Q, K, V, None, Kd, Vd, odd)
        assert torch.equal(again, out)
    full, _ = _ffi.sdpa_tree(Q, K, V, lens_t([1 << 40, s]), Kd, Vd, mask)
    none, nolse = _ffi.sdpa_tree(Q, K, V, lens_t([-5, 0]), Kd, Vd, mask, need_lse=False)
    assert torch.equal(full, out) and nolse is None
    check_tree(Q, K[:, :, :0], V[:, :, :0], [0, 0], Kd, Vd, mask, dtype, none, torch.from_numpy(
        O.sdpa_tree(f64(Q), f64(K), f64(V), [0, 0], f64(Kd), f64(Vd), mask[None].cpu().numpy())[1]))
    empty, _ = _ffi.sdpa_tree(Q, K[:, :, :0], V[:, :, :0], None, Kd, Vd, mask)            # a cache without rows
    assert torch.equal(empty, none)
    # one element off a 16-byte boundary, and rows that do not start on one
    off = torch.randn(n * hk * s * (d + 1) + 1, generator=g).to(DT[dtype]).cuda()[1:].view(n, hk, s, d + 1)[..., :d]
    out, lse = _ffi.sdpa_tree(Q, off, V, None, Kd, Vd, mask)
    check_tree(Q, off, V, None, Kd, Vd, mask, dtype, out, lse)
    # every other feature of a wider tensor: not contiguous, copied
    wide = torch.randn(n, hk, s, 2 * d, generator=g).to(DT[dtype]).cuda()[..., ::2]
    out, lse = _ffi.sdpa_tree(Q, wide, V, None, Kd, Vd, mask)
    check_tree(Q, wide, V, None, Kd, Vd, mask, dtype, out, lse)
    # a cache that several entries share (stride 0)
    one = K[:1].expand(n, hk, s, d)
    out, lse = _ffi.sdpa_tree(Q, one, V, None, Kd, Vd, mask)
    check_tree(Q, one, V, None, Kd, Vd, mask, dtype, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("h,hk,l", [(8, 8, 3), (16, 4, 12), (32, 8, 27)])
def test_tree_and_mass_many_launches_never_time_out(cuda, h, hk, l):
    """Every wait in the pipelines ends by its event: thousands of launches of uneven lengths leave the error word at zero, and
    the last result is the first one's."""
    Q, K, V, Kd, Vd, mask = tree_inputs(8, h, hk, l, 1500, 128, "bf16", seed=h)
    lens = [lens_t([(i * 331 + j * 97) % 1501 for i in range(8)]) for j in range(5)]
    first = [_ffi.sdpa_tree(Q, K, V, x, Kd, Vd, mask) for x in lens]
    ones = [_ffi.attn_mass(Q, K, f[1], kv_lens=x, is_causal=False) for f, x in zip(first, lens)]
    for _ in range(600):
        last = [_ffi.sdpa_tree(Q, K, V, x, Kd, Vd, mask) for x in lens]
        mass = [_ffi.attn_mass(Q, K, f[1], kv_lens=x, is_causal=False) for f, x in zip(first, lens)]
    assert _ffi.tc_error() == 0
    for a, b, c, d in zip(first, last, ones, mass):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(c, d)


@pytest.mark.gpu
def test_tree_with_other_value_dim(cuda):
    for d, dv, dtype in ((128, 64, "bf16"), (64, 128, "f16"), (40, 8, "bf16"), (20, 50, "f32")):
        Q, K, V, Kd, Vd, mask = tree_inputs(1, 4, 2, 5, 140, d, dtype, seed=d, dv=dv)
        out, lse = _ffi.sdpa_tree(Q, K, V, lens_t([133]), Kd, Vd, mask)
        check_tree(Q, K, V, [133], Kd, Vd, mask, dtype, out, lse)


@pytest.mark.gpu
def test_tree_of_one_node_is_decode_attention(cuda):
    """One drafted token that sees itself: what sdpa computes once the token's row is in the cache."""
    Q, K, V, Kd, Vd, _ = tree_inputs(3, 8, 2, 1, 700, 128, "bf16", seed=2)
    lens = [699, 300, 64]
    out, lse = _ffi.sdpa_tree(Q, K, V, lens_t(lens), Kd, Vd, torch.ones(1, 1, dtype=torch.bool, device="cuda"))
    for b, n in enumerate(lens):
        K[b, :, n], V[b, :, n] = Kd[b, :, 0], Vd[b, :, 0]
    want, wl = _ffi.sdpa(Q, K, V, is_causal=True, kv_lens=lens_t([n + 1 for n in lens]))
    # both round their weights and their result once: twice the distance of each from the exact value
    assert (out.float() - want.float()).abs().max() <= 4 * 2.0 ** -8 * V.float().abs().max()
    assert (lse - wl).abs().max() < 1e-4


@pytest.mark.gpu
def test_tree_offsets_beyond_32_bits(cuda):
    """A cache whose last rows lie more than 2^31 elements behind its first."""
    n, hk, s, d, l = 3, 8, 1 << 20, 128, 4
    K = torch.empty(n, hk, s, d, dtype=torch.bfloat16, device="cuda")
    V = torch.empty(n, hk, s, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    small = torch.randn(2, hk, 200, d, generator=g).bfloat16().cuda()
    K[2, :, :200], V[2, :, :200] = small[0], small[1]
    Q, _, _, Kd, Vd, mask = tree_inputs(1, 16, hk, l, 8, d, "bf16", seed=4)
    wide = lambda t: t.expand(n, *t.shape[1:])                                                  # noqa: E731
    out, lse = _ffi.sdpa_tree(wide(Q), K, V, lens_t([0, 0, 200]), wide(Kd), wide(Vd), mask)
    want, wl = _ffi.sdpa_tree(Q, small[:1], small[1:], lens_t([200]), Kd, Vd, mask)
    assert torch.allclose(out[2:].float(), want.float(), atol=4 * 2.0 ** -8 * float(want.abs().max()), rtol=0) and torch.allclose(lse[2:], wl, atol=1e-4)
    mass = _ffi.attn_mass(Q, K[2:], lse[2:].contiguous(), kv_lens=lens_t([200]), is_causal=False)
    part = _ffi.attn_mass(Q, small[:1], lse[2:].contiguous(), kv_lens=lens_t([200]), is_causal=False)
    assert torch.equal(mass[:, :, :200], part) and float(mass[:, :, 200:].abs().max()) == 0.0
    _ffi.kv_append(K, V, lens_t([0, 0, s - l]), Kd.expand(n, hk, l, d), Vd.expand(n, hk, l, d))
    assert torch.equal(K[2, :, s - l:], Kd[0]) and torch.equal(V[2, :, s - l:], Vd[0]) and torch.equal(K[1, :, :l], Kd[0])


# ------------------------------------------------------------------------------------------------
# acceptance and commit
# ------------------------------------------------------------------------------------------------
def accept_inputs(n, l, shared, seed, hit=0.75):
    g = torch.Generator().manual_seed(seed)
    par = tree_parents(1 if shared else n, l, g)
    target = torch.randint(0, 50, (n, l), generator=g)
    said = target.gather(1, par.clamp(min=0).expand(n, l))
    draft = torch.where(torch.rand(n, l, generator=g) < hit, said, torch.randint(0, 50, (n, l), generator=g))
    return par, draft, target


@pytest.mark.gpu
@pytest.mark.parametrize("n,l,shared", [(1, 1, True), (1, 2, True), (3, 8, False), (5, 33, True), (2, 128, False), (4, 129, False), (2, 1000, False)])
def test_tree_accept(cuda, n, l, shared):
    for seed, hit in ((1, 0.75), (2, 1.0), (3, 0.0)):
        par, draft, target = accept_inputs(n, l, shared, seed * 100 + l, hit)
        if hit == 1.0 and l > 2:
            par[:, l // 2] = -1                                        # a padded node and all below it take no part
        got = _ffi.tree_accept(par.cuda(), draft.cuda(), target.cuda())
        want = O.tree_accept(par.numpy(), draft.numpy(), target.numpy())
        for a, b in zip(got, want):
            assert np.array_equal(a.cpu().numpy(), b)
    chain = torch.arange(-1, l - 1)
    got = _ffi.tree_accept(chain.cuda(), target.gather(1, chain.clamp(min=0).expand(n, l)).cuda(), target.cuda())
    assert (got[1].cpu() == l).all() and (got[0].cpu() == torch.arange(l)).all() and (got[2].cpu() == target[:, -1]).all()
    assert _ffi.check_status(torch.device("cuda", 0)) == 0


@pytest.mark.gpu
def test_tree_accept_flags_parents_out_of_order(cuda):
    par = torch.tensor([[-1, 0, 3, 1, 900]])
    t = torch.zeros(1, 5, dtype=torch.int64)
    path, counts, _ = _ffi.tree_accept(par.cuda(), t.cuda(), t.cuda())
    assert path[0].tolist() == [0, 1, 3, -1, -1] and counts.tolist() == [3]
    assert _ffi.check_status(torch.device("cuda", 0)) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,dv", [("bf16", 128, 128), ("f16", 64, 40), ("f32", 36, 36), ("bf16", 33, 33), ("f32", 5, 3)])
def test_kv_append(cuda, dtype, d, dv):
    layers, g, hk, l, cap = 3, 4, 2, 6, 20
    gen = torch.Generator().manual_seed(d)
    n = layers * g
    r = lambda *sh: torch.randn(*sh, generator=gen).to(DT[dtype]).cuda()                        # noqa: E731
    K, V, Kn, Vn = r(n, hk, cap, d), r(n, hk, cap, dv), r(n, l, hk, d).transpose(1, 2), r(n, hk, l, dv)
    lens, counts = [0, 14, 7, 13], [6, 6, 0, 3]
    path = torch.stack([torch.randperm(l, generator=gen).sort().values for _ in range(g)])
    path[3] = torch.tensor([1, 4, 5, -1, -1, -1])
    nxt = torch.tensor([3, 100, 7, 50])
    pos, mass = torch.full((n, hk, cap), -7, dtype=torch.int32).cuda(), torch.ones(n, hk, cap).cuda()
    want = [x.cpu().clone() for x in (K, V, pos, mass)]
    for b in range(n):
        for t in range(counts[b % g]):
            at, row = lens[b % g] + t, int(path[b % g, t])
            want[0][b, :, at], want[1][b, :, at] = Kn[b, :, row].cpu(), Vn[b, :, row].cpu()
            want[2][b, :, at], want[3][b, :, at] = int(nxt[b % g]) + t, 0.0
    kv = lens_t(lens)
    out = _ffi.kv_append(K, V, kv, Kn, Vn, path=path.cuda(), counts=lens_t(counts), pos=pos, next_pos=nxt.cuda(), mass=mass)
    assert out.tolist() == [6, 20, 7, 16] and kv.tolist() == lens
    for a, b in zip((K, V, pos, mass), want):
        assert torch.equal(a.cpu(), b)
    assert _ffi.check_status(torch.device("cuda", 0)) == 0
    # without a path all rows go in order; without counts all of them
    out = _ffi.kv_append(K, V, lens_t([2] * g), Kn, Vn)
    assert out.tolist() == [8] * g and torch.equal(K[:, :, 2:8], Kn) and torch.equal(V[:, :, 2:8], Vn)


@pytest.mark.gpu
def test_kv_append_skips_what_does_not_fit(cuda):
    K = torch.zeros(1, 1, 4, 8, device="cuda")
    V = torch.zeros(1, 1, 4, 8, device="cuda")
    Kn = torch.arange(1.0, 4.0, device="cuda").view(1, 1, 3, 1).expand(1, 1, 3, 8).contiguous()
    out = _ffi.kv_append(K, V, lens_t([2]), Kn, Kn, path=lens_t([[2, 9, 0]]))          # row 9 does not exist, slot 4 neither
    assert out.tolist() == [4] and K[0, 0, :, 0].tolist() == [0, 0, 3, 0]
    assert _ffi.check_status(torch.device("cuda", 0)) == 1
    out = _ffi.kv_append(K, V, lens_t([-1]), Kn, Kn, counts=lens_t([2]))               # slot -1 is skipped
    assert out.tolist() == [1] and K[0, 0, :, 0].tolist() == [2, 0, 3, 0]
    assert _ffi.check_status(torch.device("cuda", 0)) == 1


# ------------------------------------------------------------------------------------------------
# attention mass
# ------------------------------------------------------------------------------------------------
def check_mass(Q, K, lse, lens, limits, mass, out, scale=None):
    n, l, s = Q.shape[0], Q.shape[2], K.shape[2]
    base = f64(mass) if mass is not None else np.zeros((n, K.shape[1], s))
    ref, reach = O.attn_mass(f64(Q), f64(K), f64(lse), lens, limits, base, scale)
    rows = Q.shape[1] // K.shape[1] * l
    # each weight as in the attention test; its lse is an input, scaled to the log2 domain (2^-23 of it); a sum of `rows`
    big = float(np.abs(f64(lse))[np.isfinite(f64(lse))].max(initial=0.0))
    rel = 2 * (Q.shape[3] + 8) * 2.0 ** -24 * reach + 2.0 ** -20 + 2.0 ** -22 * big + rows * 2.0 ** -24
    tol = rel * np.abs(ref - base) + 2.0 ** -23 * np.abs(ref) + 2.0 ** -40
    err = np.abs(f64(out) - ref)
    assert (err <= tol).all(), (err / tol).max()


MASS_CASES = [
    # n, h, hk, l, s, d, lens, dtype
    (1, 4, 4, 1, 128, 128, [128], "bf16"),
    (3, 8, 2, 1, 300, 128, [300, 1, 129], "f16"),
    (2, 8, 2, 5, 131, 128, [130, 77], "bf16"),
    (1, 8, 2, 64, 257, 128, [257], "f16"),
    (1, 6, 2, 100, 300, 128, [290], "bf16"),            # three heads per KV head, several tiles of rows
    (1, 7, 1, 40, 140, 64, [140], "bf16"),
    (1, 2, 2, 200, 200, 64, [200], "f16"),
    (1, 2, 1, 300, 300, 128, [300], "bf16"),            # a prompt
    (2, 4, 2, 20, 150, 80, [149, 20], "bf16"),
    (1, 4, 2, 9, 70, 40, [66], "f16"),
    (1, 2, 2, 9, 70, 33, [70], "bf16"),
    (2, 4, 2, 17, 150, 128, [149, 17], "f32"),
    (1, 2, 1, 5, 90, 300, [88], "f32"),
    (1, 160, 1, 2, 70, 128, [65], "bf16"),
    (5, 4, 2, 3, 600, 128, [600, 3, 64, 500, 599], "bf16"),
    (300, 2, 1, 2, 40, 64, [2 + i % 39 for i in range(300)], "bf16"),           # more key counts than the kernel keeps on chip
    (3, 12, 3, 120, 400, 128, [400, 120, 333], "f16"),                           # few row tiles, many items
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", MASS_CASES, ids=lambda c: "-".join(str(x) for x in c[:6] + c[7:] + (c[6][:3],)).replace(" ", ""))
def test_attn_mass(cuda, case, causal):
    n, h, hk, l, s, d, lens, dtype = case
    g = torch.Generator().manual_seed(l * 100 + s)
    Q, K = (torch.randn(*sh, generator=g).to(DT[dtype]).cuda() for sh in ((n, h, l, d), (n, hk, s, d)))
    mass = torch.rand(n, hk, s, generator=g).cuda()
    lim = [[(i + 1 + lens[b] - l) if causal else lens[b] for i in range(l)] for b in range(n)]
    # the lse a full softmax would have left, and one row that saw nothing, one that is left out
    x = torch.einsum("nhld,nhsd->nhls", Q.double(), K.double().repeat_interleave(h // hk, 1)) * d ** -0.5
    seen = torch.arange(s).cuda() < torch.tensor(lim).cuda()[:, None, :, None]
    lse = x.masked_fill(~seen, -float("inf")).logsumexp(-1).float()
    if l > 2:
        lse[0, 0, 1], lse[0, 1, 2] = float("inf"), -float("inf")
    K = K.clone()
    for b in range(n):
        K[b, :, lens[b]:] = float("nan")                               # behind the count: never looked at
    out = _ffi.attn_mass(Q, K, lse, kv_lens=lens_t(lens), is_causal=causal, mass=mass)
    check_mass(Q, K, lse, lens, lim, mass, out)
    for b in range(n):
        assert torch.equal(out[b, :, lens[b]:], mass[b, :, lens[b]:])
    again = mass.clone()
    assert _ffi.attn_mass(Q, K, lse, kv_lens=lens_t(lens), is_causal=causal, mass=again, out=again) is again
    assert torch.equal(again, out)                                     # in place, and no sum depends on timing
    zero = _ffi.attn_mass(Q, K, lse, kv_lens=lens_t(lens), is_causal=causal)
    check_mass(Q, K, lse, lens, lim, None, zero)
    if l <= 2 and (causal is False or min(lens) >= l):
        # the weights of a row sum to one, so a head's share of the mass is its rows
        assert abs(float(zero.sum()) - n * h * l) < 1e-4 * n * h * l
    assert _ffi.tc_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 64)])
def test_attn_mass_row_limits_layers_views_and_scale(cuda, dtype, d):
    layers, g, h, hk, l, s = 2, 2, 4, 2, 6, 140
    n = layers * g
    gen = torch.Generator().manual_seed(8)
    qkv = torch.randn(n * l, (h + 2 * hk) * d, generator=gen).to(DT[dtype]).cuda()
    W = qkv.shape[1]
    Q = qkv.as_strided((n, h, l, d), (l * W, d, W, 1))
    K = torch.randn(n, hk, s + 7, d, generator=gen).to(DT[dtype]).cuda()[:, :, 7:]
    lse = torch.randn(n, h, l, generator=gen).cuda() + 4
    lens, lim = [140, 99], [[0, 3, 1 << 40, 64, -2, 99], [99, 98, 1, 0, 140, 65]]
    for scale in (None, 0.3, -0.1):
        out = _ffi.attn_mass(Q, K, lse, kv_lens=lens_t(lens), q_lens=lens_t(lim), scale=scale)
        check_mass(Q, K, lse, lens * layers, lim * layers, None, out, scale)
    out = _ffi.attn_mass(Q, K, lse, is_causal=True)
    check_mass(Q, K, lse, [s] * n, [[i + 1 + s - l for i in range(l)]] * n, None, out)
    off = torch.randn(n * hk * s * (d + 1) + 1, generator=gen).to(DT[dtype]).cuda()[1:].view(n, hk, s, d + 1)[..., :d]
    out = _ffi.attn_mass(Q, off, lse, is_causal=False)
    check_mass(Q, off, lse, [s] * n, [[s] * l] * n, None, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,hk,l,s,d", [(3, 16, 2, 64, 98, 64), (1, 8, 8, 33, 397, 128), (1, 2, 1, 40, 70, 256), (1, 2, 2, 7, 45, 300),
                                          (2, 4, 2, 9, 33, 512), (1, 2, 1, 20, 40, 513), (1, 2, 1, 35, 65, 1000), (1, 1, 1, 1, 2, 1024),
                                          (1, 4, 2, 16, 300, 250), (150, 4, 4, 9, 600, 62), (2, 40, 1, 1, 130, 37)])
def test_attn_mass_row_counts_and_wide_heads(cuda, dtype, n, h, hk, l, s, d):
    """Few keys under many rows, many keys under few, heads up to the widest that is taken."""
    g = torch.Generator().manual_seed(l + s)
    Q, K = (torch.randn(*sh, generator=g).to(DT[dtype]).cuda() for sh in ((n, h, l, d), (n, hk, s, d)))
    lens = [s - b % 5 for b in range(n)]
    x = torch.einsum("nhld,nhsd->nhls", Q.double(), K.double().repeat_interleave(h // hk, 1)) * d ** -0.5
    lim = [[i + 1 + lens[b] - l for i in range(l)] for b in range(n)]
    seen = torch.arange(s).cuda() < torch.tensor(lim).cuda()[:, None, :, None]
    lse = x.masked_fill(~seen, -float("inf")).logsumexp(-1).float()
    mass = torch.rand(n, hk, s, generator=g).cuda()
    out = _ffi.attn_mass(Q, K, lse, mass=mass, kv_lens=lens_t(lens), is_causal=True)
    check_mass(Q, K, lse, lens, lim, mass, out)


@pytest.mark.gpu
def test_attn_mass_spreads_nan_only_where_it_belongs(cuda):
    g = torch.Generator().manual_seed(8)
    Q, K = torch.randn(1, 2, 4, 128, generator=g).bfloat16().cuda(), torch.randn(1, 2, 130, 128, generator=g).bfloat16().cuda()
    lse = torch.full((1, 2, 4), 5.0, device="cuda")
    K[0, 0, 17, 3] = float("nan")
    out = _ffi.attn_mass(Q, K, lse, is_causal=False)
    bad = torch.zeros(1, 2, 130, dtype=torch.bool)
    bad[0, 0, 17] = True
    assert torch.equal(torch.isnan(out).cpu(), bad)
    K[0, 0, 17, 3] = 0
    lse[0, 1, 2] = float("nan")
    out = _ffi.attn_mass(Q, K, lse, q_lens=lens_t([[130, 130, 9, 130]]))
    bad = torch.zeros(1, 2, 130, dtype=torch.bool)
    bad[0, 1, :9] = True
    assert torch.equal(torch.isnan(out).cpu(), bad)


# ------------------------------------------------------------------------------------------------
# eviction
# ------------------------------------------------------------------------------------------------
def check_evict(K, V, mass, lens, budget, *, pos=None, next_pos=None, sinks=0, recent=0):
    n, hk, cap, _ = K.shape
    g = len(lens)
    want = [K.cpu().clone(), V.cpu().clone(), torch.zeros(n, hk, cap), torch.full((n, hk, cap), -1, dtype=torch.int32),
            torch.full((n, hk, budget), -1, dtype=torch.int32)]
    before = [t.clone() for t in (mass,) + ((pos,) if pos is not None else ())]
    m, p = mass.cpu().numpy(), (pos.cpu().numpy() if pos is not None else np.broadcast_to(np.arange(cap), (n, hk, cap)))
    k0, v0 = want[0].clone(), want[1].clone()
    for b in range(n):
        length = min(max(lens[b % g], 0), cap)
        for i in range(hk):
            src = torch.tensor(O.kv_evict_map(m[b, i], p[b, i], length, next_pos[b % g] if next_pos else length, budget, sinks, recent), dtype=torch.long)
            k = len(src)
            want[0][b, i, :k], want[1][b, i, :k] = k0[b, i, src], v0[b, i, src]
            want[2][b, i, :k], want[3][b, i, :k], want[4][b, i, :k] = torch.from_numpy(m[b, i][src.numpy()]), torch.from_numpy(p[b, i][src.numpy()]).int(), src.int()
    got = _ffi.kv_evict(K, V, mass, lens_t(lens), budget, pos=pos, next_pos=lens_t(next_pos) if next_pos else None, sinks=sinks, recent=recent)
    assert got[0].tolist() == [min(min(max(x, 0), cap), budget) for x in lens]
    assert torch.equal(got[3].cpu(), want[4]) and torch.equal(got[2].cpu(), want[3])
    assert np.array_equal(got[1].cpu().numpy(), want[2].numpy(), equal_nan=True)
    assert torch.equal(K.cpu().float().nan_to_num(7), want[0].float().nan_to_num(7)) and torch.equal(V.cpu(), want[1])
    for a, b in zip((mass,) + ((pos,) if pos is not None else ()), before):
        assert torch.equal(a.nan_to_num(3.0) if a.is_floating_point() else a, b.nan_to_num(3.0) if b.is_floating_point() else b)
    again = _ffi.kv_evict(K, V, mass, lens_t(lens), budget, pos=pos, next_pos=lens_t(next_pos) if next_pos else None, sinks=sinks, recent=recent)
    assert torch.equal(again[3], got[3]) and torch.equal(V.cpu(), want[1])             # the call may be repeated
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("lens,cap,budget,sinks,recent", [
    ([5], 5, 1, 0, 0), ([5], 5, 5, 2, 3), ([33], 40, 32, 0, 0), ([1, 0, -3], 40, 7, 0, 2), ([64, 1 << 40], 64, 20, 4, 8),
    ([1000, 1024, 1025], 1100, 500, 4, 100), ([2050, 31], 2100, 2049, 1, 1), ([5000], 5000, 100, 10, 90), ([4097, 4096], 4100, 3000, 0, 0),
    ([33000], 33000, 16000, 4, 64), ([300000], 300000, 200000, 4, 64), ([400000], 400000, 1000, 4, 64),       # keys kept in shared memory over a cluster, and too many for it
])
def test_kv_evict(cuda, lens, cap, budget, sinks, recent):
    g = torch.Generator().manual_seed(cap + budget)
    n, hk, d = len(lens) * 2, 2, 8
    K, V = torch.randn(n, hk, cap, d, generator=g).bfloat16().cuda(), torch.randn(n, hk, cap, d, generator=g).bfloat16().cuda()
    mass = torch.exp(2 * torch.randn(n, hk, cap, generator=g)).cuda()
    check_evict(K, V, mass, lens, budget, sinks=sinks, recent=recent)


@pytest.mark.gpu
def test_kv_evict_ties_specials_and_positions(cuda):
    g = torch.Generator().manual_seed(6)
    n, hk, cap, d = 6, 1, 300, 4
    K, V = torch.randn(n, hk, cap, d, generator=g).cuda(), torch.randn(n, hk, cap, d, generator=g).cuda()
    mass = torch.randint(0, 4, (n, hk, cap), generator=g).float()
    mass[1] = 1.0                                                      # all the same
    mass[2] = torch.where(torch.rand(1, cap, generator=g) < 0.5, -0.0, 0.0)
    mass[3, :, ::7], mass[3, :, 3::7], mass[3, :, 5::7] = float("nan"), float("inf"), -float("inf")
    mass[4] = torch.randn(1, cap, generator=g)                         # negative weights too
    mass[5, :, :] = torch.tensor([1e-45, 3e-45, 1e-38, 2e-38]).repeat(75)      # denormals
    lens = [300, 299, 280, 300, 256, 300]
    for budget in (1, 64, 150, 255):
        check_evict(K.clone(), V.clone(), mass.cuda(), lens, budget, sinks=0, recent=min(budget, 30))
    # positions out of order, as earlier evictions leave them; more protected slots than the budget holds
    pos = torch.stack([torch.randperm(1000, generator=g)[:cap] for _ in range(n)]).view(n, 1, cap).int()
    check_evict(K.clone(), V.clone(), mass.cuda(), lens, 100, pos=pos.cuda(), next_pos=[1000] * n, sinks=20, recent=60)
    check_evict(K.clone(), V.clone(), mass.cuda(), lens, 20, pos=pos.cuda(), next_pos=[900] * n, sinks=10, recent=10)
    pos[:] = 5
    check_evict(K.clone(), V.clone(), mass.cuda(), lens, 40, pos=pos.cuda(), next_pos=[900] * n, sinks=10, recent=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,dv", [("bf16", 128, 128), ("f16", 40, 64), ("bf16", 33, 7), ("f32", 6, 6)])
def test_kv_evict_layouts(cuda, dtype, d, dv):
    """Head dims, strided caches, NaN payloads, one key count for several layers."""
    g = torch.Generator().manual_seed(d)
    base = torch.randn(2, 2, 200, 3, d, generator=g).to(DT[dtype]).cuda()
    K, V = base.permute(0, 3, 2, 1, 4).reshape(2, 3, 400, d)[:, :, 100:350], torch.randn(2, 3, 250, dv, generator=g).to(DT[dtype]).cuda()
    V = V.transpose(1, 2).contiguous().transpose(1, 2)                 # (n, cap, h, d) in memory
    K[:, :, 240, 0] = float("nan")
    check_evict(K, V, torch.rand(2, 3, 250, generator=g).cuda(), [245], 100, sinks=2, recent=10)


# ------------------------------------------------------------------------------------------------
# the operators together
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_verified_steps_equal_token_by_token_decoding(cuda):
    """A chain verified as a tree, accepted and committed leaves the cache a token-by-token loop leaves; evicting down to a
    budget keeps exactly the slots with the most weight, and attention over them equals attention over the kept keys."""
    n, h, hk, l, cap, d = 2, 8, 2, 5, 96, 128
    Q, K, V, Kd, Vd, _ = tree_inputs(n, h, hk, l, cap, d, "bf16", seed=21)
    lens = lens_t([40, 33])
    par = torch.tensor([-1, 0, 0, 1, 3])
    mask = ancestors(par[None])[0].cuda()
    out, lse = _ffi.sdpa_tree(Q, K, V, lens, Kd, Vd, mask)
    target = torch.randint(0, 9, (n, l), generator=torch.Generator().manual_seed(0))
    draft = target.gather(1, par.clamp(min=0).expand(n, l)).clone()
    draft[1, 3] += 1                                                   # the second sequence stops after node 1 (or 2)
    path, counts, _ = _ffi.tree_accept(par.cuda(), draft.cuda(), target.cuda())
    assert path.tolist() == [[0, 1, 3, 4, -1], [0, 1, -1, -1, -1]] and counts.tolist() == [4, 2]
    pos, mass = torch.arange(cap, dtype=torch.int32).expand(n, hk, cap).contiguous().cuda(), torch.zeros(n, hk, cap).cuda()
    new = _ffi.kv_append(K, V, lens, Kd, Vd, path=path, counts=counts, pos=pos, next_pos=lens, mass=mass)
    assert new.tolist() == [44, 35]
    # row 4 of the first sequence saw the cache and nodes 0, 1, 3, 4: what decoding token by token sees
    one, one_lse = _ffi.sdpa(Q[:1, :, 4:5], K[:1], V[:1], is_causal=True, kv_lens=new[:1])
    assert (out[:1, :, 4:5].float() - one.float()).abs().max() <= 4 * 2.0 ** -8 * V.float().abs().max()
    assert (lse[:1, :, 4:5] - one_lse).abs().max() < 1e-4
    # weight of the accepted rows: row path[t] counts for lens + t + 1 keys, the others for none
    q_lens = torch.zeros(n, l, dtype=torch.int64, device="cuda")
    for b in range(n):
        for t in range(int(counts[b])):
            q_lens[b, path[b, t]] = lens[b] + t + 1
    mass = _ffi.attn_mass(Q, K, lse, kv_lens=new, q_lens=q_lens, mass=mass, out=mass)
    # each accepted row spreads a weight of one per head, all of it over keys in the cache now
    assert torch.allclose(mass.sum(-1), (counts * (h // hk)).float()[:, None].expand(n, hk), atol=2e-3)
    budget = 30
    before, values = K.clone(), V.clone()
    kept, mass, pos, src = _ffi.kv_evict(K, V, mass, new, budget, pos=pos, next_pos=new, sinks=2, recent=8)
    assert kept.tolist() == [30, 30] and (pos[:, :, :30] == src).all()
    for b in range(n):
        for i in range(hk):
            rows = set(src[b, i].tolist())
            assert {0, 1} <= rows and set(range(int(new[b]) - 8, int(new[b]))) <= rows and len(rows) == 30
            assert torch.equal(K[b, i, :30], before[b, i, src[b, i].long()])
    after, al = _ffi.sdpa(Q[:, :, :1], K, V, is_causal=True, kv_lens=kept)
    order = src.long().sort(-1).values[..., None].expand(n, hk, budget, d)
    want, wl = _ffi.sdpa(Q[:, :, :1], before.gather(2, order), values.gather(2, order), is_causal=True)
    assert (after.float() - want.float()).abs().max() <= 4 * 2.0 ** -8 * V.float().abs().max() and (al - wl).abs().max() < 1e-4


@pytest.mark.gpu
def test_calls_on_a_side_stream_first_captured_and_without_launch_overlap(cuda):
    """A first use inside a capture on a fresh stream, replayed on changed inputs; and the same calls with programmatic launches
    off."""
    n, h, hk, l, s, d = 2, 8, 2, 5, 900, 128
    Q, K, V, Kd, Vd, mask = tree_inputs(n, h, hk, l, s, d, "bf16", seed=41)
    par, draft, target = (t.cuda() for t in accept_inputs(n, l, True, 7))
    lens = lens_t([700, 650])
    side = torch.cuda.Stream()

    def step():
        out, lse = _ffi.sdpa_tree(Q, K, V, lens, Kd, Vd, mask)
        path, counts, nxt = _ffi.tree_accept(par, draft, target)
        new = _ffi.kv_append(K, V, lens, Kd, Vd, path=path, counts=counts)
        return out, lse, path, counts, nxt, new, _ffi.attn_mass(Q, K, lse, kv_lens=lens, is_causal=False)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        got = step()
    for k in range(3):
        Q.copy_(torch.randn(Q.shape, generator=torch.Generator().manual_seed(k)))
        lens.copy_(lens_t([700 - k, 650 - 64 * k]))
        gr.replay()
        torch.cuda.synchronize()
        have = [t.clone() for t in got]
        want = step()
        old = _ffi.set_pdl(False)
        plain = step()
        _ffi.set_pdl(old)
        for a, b, c in zip(have, want, plain):
            assert torch.equal(a, b) and torch.equal(a, c)
    del gr


@pytest.mark.gpu
def test_captured_replayed_and_on_several_streams(cuda):
    """Two graphs of the same calls, replayed on two streams at once, and an eager call between them."""
    n, h, hk, l, s, d = 2, 8, 2, 6, 3000, 128
    Q, K, V, Kd, Vd, mask = tree_inputs(n, h, hk, l, s, d, "bf16", seed=31)
    lens = lens_t([2900, 1500])
    ev = torch.randn(2, n, hk, s, d, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()

    def step(q, cache):
        out, lse = _ffi.sdpa_tree(q, K, V, lens, Kd, Vd, mask)
        mass = _ffi.attn_mass(q, K, lse, kv_lens=lens, is_causal=False)
        return (out, lse, mass) + _ffi.kv_evict(cache[0], cache[1], mass, lens, 1000, sinks=4, recent=100)
    q2 = Q.flip(0).contiguous()
    ref1, ref2 = [t.clone() for t in step(Q, ev.clone())], [t.clone() for t in step(q2, ev.clone())]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    caches = [ev.clone(), ev.clone()]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for st, q, c in zip(streams, (Q, q2), caches):
        with torch.cuda.stream(st):
            step(q, c)                                                 # warm-up on the stream of the capture
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            outs.append(step(q, c))
        graphs.append(gr)
    for _ in range(5):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        eager = step(Q, ev.clone())
        torch.cuda.synchronize()
        for got, ref in zip(outs + [eager], (ref1, ref2, ref1)):
            for a, b in zip(got, ref):
                assert torch.equal(a, b)
    del graphs
