"""Verified trees and evictions of a tensor-parallel decoder, on CPU ranks (gloo, world size 2): plain torch in 64 bits stands in
for the kernels, what is under test is the decoder's sharding of heads, caches, weight and vocabulary around them."""
import datetime
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from kuillm_b200 import decoder as D
from oracle import kuiops_oracle as O


class Plain:
    """The calls that the decoder makes of the library, from their definitions."""

    @staticmethod
    def embedding(w, ids):
        return w[ids].clone()

    @staticmethod
    def rmsnorm(x, w, eps, residual=None):
        if residual is not None:
            residual += x
            x = residual
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w

    @staticmethod
    def gemm(a, b, trans_b=True, out=None):
        y = a @ b.t()
        return y if out is None else out.copy_(y)

    @staticmethod
    def gemm_swiglu(a, wgu):
        y = a @ wgu.t()
        return torch.nn.functional.silu(y[:, 0::2]) * y[:, 1::2]

    @staticmethod
    def rope_qkv(qkv, hq, hk, hd, positions, theta, k_cache=None, v_cache=None, rows_per_seq=1):
        rows = qkv.shape[0]
        t = qkv.view(rows, hq + 2 * hk, hd)
        ang = positions.double()[:, None] * theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        a, b = t[:, :hq + hk, :hd // 2].clone(), t[:, :hq + hk, hd // 2:].clone()
        t[:, :hq + hk, :hd // 2], t[:, :hq + hk, hd // 2:] = a * c - b * s, b * c + a * s
        if k_cache is not None:
            for r in range(rows):
                k_cache[r // rows_per_seq, :, positions[r]] = t[r, hq:hq + hk]
                v_cache[r // rows_per_seq, :, positions[r]] = t[r, hq + hk:]

    @staticmethod
    def sdpa(q, k, v, is_causal, need_lse, out, kv_lens=None):
        l, s, g = q.shape[2], k.shape[2], q.shape[1] // k.shape[1]
        x = q @ k.repeat_interleave(g, 1).transpose(2, 3) * q.shape[3] ** -0.5
        x = x.masked_fill(~torch.ones(l, s, dtype=torch.bool).tril(s - l), -float("inf"))
        out.copy_(torch.softmax(x, -1) @ v.repeat_interleave(g, 1))
        return out, x.logsumexp(-1)

    @staticmethod
    def sdpa_tree(q, k, v, kv_lens, kd, vd, mask, need_lse, out):
        y, lse = O.sdpa_tree(q, k, v, kv_lens.tolist(), kd, vd, mask[None].numpy())[:2]
        return out.copy_(torch.from_numpy(y)), torch.from_numpy(lse)

    @staticmethod
    def tree_accept(parents, draft, target):
        return [torch.from_numpy(x) for x in O.tree_accept(parents[None].numpy(), draft.numpy(), target.numpy())]

    @staticmethod
    def kv_append(K, V, kv_lens, kn, vn, path, counts, pos, next_pos, mass):
        g = len(kv_lens)
        for b in range(K.shape[0]):
            for t in range(int(counts[b % g])):
                at, row = int(kv_lens[b % g]) + t, int(path[b % g, t])
                K[b, :, at], V[b, :, at] = kn[b, :, row], vn[b, :, row]
                pos[b, :, at] = int(next_pos[b % g]) + t
                if mass is not None:
                    mass[b, :, at] = 0
        return kv_lens + counts

    @staticmethod
    def attn_mass(q, k, lse, kv_lens, mass, out, q_lens=None, is_causal=True):
        n, g, l = q.shape[0], len(kv_lens), q.shape[2]
        lens = [int(kv_lens[b % g]) for b in range(n)]
        lim = [q_lens[b % g].tolist() if q_lens is not None else [i + 1 + lens[b] - l for i in range(l)] for b in range(n)]
        return out.copy_(torch.from_numpy(O.attn_mass(q, k, lse, lens, lim, mass)[0]))

    @staticmethod
    def kv_evict(K, V, mass, kv_lens, budget, pos, next_pos, sinks, recent):
        n, hk, cap, _ = K.shape
        g = len(kv_lens)
        src_all = torch.full((n, hk, budget), -1, dtype=torch.int32)
        mass_out, pos_out = torch.zeros_like(mass), torch.full_like(pos, -1)
        for b in range(n):
            for i in range(hk):
                src = torch.tensor(O.kv_evict_map(mass[b, i].numpy(), pos[b, i].numpy(), int(kv_lens[b % g]), int(next_pos[b % g]), budget, sinks, recent))
                k = len(src)
                K[b, i, :k], V[b, i, :k] = K[b, i, src], V[b, i, src]
                mass_out[b, i, :k], pos_out[b, i, :k], src_all[b, i, :k] = mass[b, i, src], pos[b, i, src], src.int()
        return kv_lens.clamp(max=budget), mass_out, pos_out, src_all

    @staticmethod
    def argmax_lastdim(x):
        return x.argmax(-1)

    @staticmethod
    def gather(x, dim, idx):
        return x.gather(dim, idx)

    @staticmethod
    def add_i64_(x, v):
        return x.add_(v)

    @staticmethod
    def index(x, dim, idx):
        return x.index_select(dim, idx[0])


def _run(rank, size):
    """Everything a rank knows after a prompt, trees, an eviction and another tree."""
    cfg = D.DecoderConfig(n_layers=2, d_model=32, n_heads=8, n_kv_heads=4, head_dim=8, d_ff=48, vocab=40, dtype=torch.float64)
    dec = D.Decoder(cfg, device="cpu", seed=3, tp_rank=rank, tp_size=size, init_std=0.4)
    dec.fold_norm = False
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 40, (2, 9), generator=g)
    dec.alloc_cache(2, 24, track_mass=True, window=4)
    last = dec.next_token(dec.prefill(ids, local_logits=True))
    tree = D.TreePlan([-1, 0, 0, 1, 1, 4], device="cpu")
    seen = []
    for step in range(4):
        if step == 3:
            dec.evict(8, sinks=1, recent=3)
        tokens = torch.cat([last[:, None], torch.randint(0, 40, (2, 5), generator=g)], 1)
        if step == 1:                              # drafts that are right: what the model says after the root, on one branch
            probe = dec.next_token(_score_root(dec, last))
            tokens[:, 1] = probe
        path, counts, last, logits = dec.verify(tokens, tree, return_logits=True)
        seen += [path, counts, last, dec._full_logits(logits.reshape(12, -1))]
    heads = lambda t: t.reshape(2, 2, dec.hk, 24, -1)                                             # noqa: E731
    return seen + [dec.kv_lens, dec.next_pos], [heads(x) for x in (dec.k_cache, dec.v_cache, dec.mass, dec.slot_pos)]


def _score_root(dec, last):
    """The logits after the root, from a tree of one node on a copy of the state."""
    keep = {k: getattr(dec, k) for k in ("k_cache", "v_cache", "mass", "kv_lens", "next_pos", "slot_pos", "_used")}
    for k in ("k_cache", "v_cache", "mass", "slot_pos"):
        setattr(dec, k, keep[k].clone())
    logits = dec.verify(last[:, None], D.TreePlan.chain(1, device="cpu"), return_logits=True)[3]
    for k, v in keep.items():
        setattr(dec, k, v)
    return logits.reshape(2, -1)


def _worker(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    D._ffi = Plain
    dist.init_process_group("gloo", rank=rank, world_size=2, timeout=datetime.timedelta(seconds=60))
    gather = dist.all_gather_into_tensor           # this backend takes flat tensors
    dist.all_gather_into_tensor = lambda out, x, group=None: gather(out.view(-1), x.reshape(-1), group=group)
    try:
        got, mine = _run(rank, 2)
        want, whole = _run(0, 1)
        for a, b in zip(got, want):
            if a.is_floating_point():
                assert torch.allclose(a, b, atol=1e-9, rtol=1e-9)
            else:
                assert torch.equal(a, b), (a, b)
        for a, b in zip(mine, whole):              # this rank's heads
            assert torch.allclose(a.double(), b[:, :, rank * 2:rank * 2 + 2].double(), atol=1e-9, rtol=1e-9)
        counts = [x for x in want[1::4][:4]]
        assert int(counts[1].min()) >= 2           # the right draft was accepted
        out.put("same")
    except Exception as e:                         # noqa: BLE001 - the parent reports it
        out.put(repr(e))
    dist.destroy_process_group()


def test_two_ranks_verify_and_evict_like_one():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    said = [q.get(timeout=180) for _ in procs]
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    assert said == ["same", "same"]
