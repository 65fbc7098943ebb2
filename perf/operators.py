"""The performance cases of the adapter and load-balance operators.

  lora     adapters of many requests beside a resident quantized projection:
           coli_hip_lora_gemm_dev. y[s] = W x[s] + scale_a B_a (A_a x[s]), a the
           row's adapter slot (outside the bank: none)
  step     one tuning step of the adapters on one projection: the changed
           adapters into the bank (coli_hip_lora_set_dev), forward, and the
           gradients of the input and of every adapter (coli_hip_lora_grad_dev)
  gemm_t   the input gradient of a resident projection, dx = dy W:
           coli_hip_gemm_t_dev
  balance  per-expert counts and the balance loss of routed rows, by sequence
           (coli_hip_balance_dev), and where "grad" says so the gradient of the
           router's logits (coli_hip_balance_grad_dev)

Weights are uniform nibbles / e2m1 codes, int4 scales |N(0, 0.01)| in fp16
values, e8m0 bytes 119..123. A request is a run of consecutive rows with one
adapter; one in eight requests has none. Ranks vary between adapters.
"""
import ctypes as C
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
DTYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}


def _lora(kind, fmt, I, O, S, requests, slots, rank, dtype, **kw):
    return dict(dict(kind=kind, fmt=fmt, I=I, O=O, S=S, requests=requests, slots=slots, rank=rank, dtype=dtype), **kw)


def _gemm_t(fmt, I, O, S, **kw):
    return dict(dict(kind="gemm_t", fmt=fmt, I=I, O=O, S=S), **kw)


def _balance(T, E, K, mode, seqs, grad, **kw):
    return dict(dict(kind="balance", T=T, E=E, K=K, mode=mode, seqs=seqs, grad=grad), **kw)


def listed():
    return [
        # one token through a small expert-sized projection with its adapter: latency alone
        _lora("lora", "int4", 2048, 1024, 1, 1, 4, 8, "f16", name="lora_token_small_int4"),
        # one token through a feed-forward up projection
        _lora("lora", "int4", 4096, 14336, 1, 1, 8, 16, "bf16", name="lora_token_int4"),
        # a decode batch: sixteen requests, each with an adapter of its own
        _lora("lora", "mxfp4", 7168, 2048, 16, 16, 32, 32, "bf16", name="lora_batch16_mxfp4"),
        # prompts of six requests in one prefill chunk, large adapters
        _lora("lora", "int4", 14336, 4096, 1024, 6, 4, 64, "bf16", name="lora_prefill1024_int4"),
        # a tuning step on a ragged projection and a short batch, f32 adapters
        _lora("step", "int4", 1000, 999, 37, 3, 2, 5, "f32", name="step_ragged37_int4"),
        # a tuning step of one adapter on a wide expert-sized projection
        _lora("step", "mxfp4", 7168, 2048, 512, 1, 1, 16, "f32", name="step_512_mxfp4"),
        # the largest: two adapters tuned in one batch on a feed-forward projection
        _lora("step", "int4", 4096, 14336, 2048, 4, 2, 32, "bf16", name="step_2048_int4"),
        # the gradient that passes through a frozen projection: a few rows, a batch
        _gemm_t("mxfp4", 7168, 2048, 16, name="gemm_t_16_mxfp4"),
        _gemm_t("int4", 4096, 14336, 512, name="gemm_t_512_int4"),
        # expert counts and balance of one decode batch (monitoring while serving)
        _balance(64, 64, 8, 0, 1, False, name="balance_serve64"),
        # a training batch of ragged sequences, sigmoid scores
        _balance(8192, 256, 8, 2, 16, True, name="balance_train8192"),
        # the largest batch, sqrt-softplus scores, many sequences
        _balance(65536, 384, 8, 3, 64, True, name="balance_train65536"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi):
    """A matrix dimension, log-uniform: mostly multiples of 128, some of 16, some odd."""
    step = rng.choice((128, 128, 16, 1))
    return max(step, int(round(_log(rng, lo, hi) / step)) * step)


def draw(rng):
    """One more case of the listed cases' ranges."""
    while True:
        kind = rng.choice(("lora", "lora", "step", "step", "gemm_t", "balance"))
        fmt = rng.choice(("int4", "mxfp4"))
        S = int(round(_log(rng, 1, 2048)))
        if kind == "balance":
            T = int(round(_log(rng, 1, 65536)))
            E = int(round(_log(rng, 8, 512)))
            c = _balance(T, E, rng.choice((1, 2, 6, 8)), rng.choice((0, 1, 2, 3)), int(round(_log(rng, 1, 64))),
                         rng.choice((True, False)))
        elif kind == "gemm_t":
            c = _gemm_t(fmt, _size(rng, 256, 14336), _size(rng, 256, 14336), S)
        else:
            requests = min(S, int(round(_log(rng, 1, 32))))
            c = _lora(kind, fmt, _size(rng, 256, 14336), _size(rng, 256, 14336), S, requests,
                      int(round(_log(rng, 1, 32 if kind == "lora" else 4))), int(round(_log(rng, 1, 64))),
                      rng.choice(("f32", "f16", "bf16")))
        if work(c)["flops"] <= 4.8e11 and c.get("I", 1) * c.get("O", 1) <= 6e7:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed, i):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1_000_003 + i * 7919 + 1) % (1 << 62))
    return g


def _weights(c, seed):
    """Nibbles [O, ceil(I / 2)] and group scales [O, ceil(I / 32)] (f32 of fp16 values, or e8m0 bytes)."""
    O, I = c["O"], c["I"]
    q = torch.randint(0, 256, (O, (I + 1) // 2), dtype=torch.uint8, device="cuda", generator=_gen(seed, 0))
    if c["fmt"] == "mxfp4":
        return q, torch.randint(119, 124, (O, (I + 31) // 32), dtype=torch.uint8, device="cuda", generator=_gen(seed, 1))
    s = (torch.randn(O, (I + 31) // 32, device="cuda", generator=_gen(seed, 1)) * 0.01).abs()
    return q, s.half().float()


def _ranks(c):
    """Rank of each slot: the largest first, others down to half of it."""
    r = c["rank"]
    return [r - (s * 5) % (r // 2 + 1) for s in range(c["slots"])]


def _adapters(c, seed):
    """A [slots, rank, I] and B [slots, O, rank], zero beyond a slot's rank, and scales [slots]."""
    g = _gen(seed, 2)
    ranks = torch.tensor(_ranks(c), device="cuda")
    live = torch.arange(c["rank"], device="cuda")[None, :] < ranks[:, None]
    a = torch.randn(c["slots"], c["rank"], c["I"], device="cuda", generator=g) / math.sqrt(c["I"])
    b = torch.randn(c["slots"], c["O"], c["rank"], device="cuda", generator=g) / math.sqrt(c["rank"])
    dt = DTYPES[c["dtype"]][1]
    scales = 0.5 + torch.rand(c["slots"], device="cuda", generator=g)
    return (a * live[:, :, None]).to(dt), (b * live[:, None, :]).to(dt), scales


def _slots(c, seed):
    """The rows' adapter slots: consecutive rows of a request share one; one request in eight has none."""
    g = _gen(seed, 3)
    n = c["requests"]
    slot = torch.randint(0, c["slots"], (n,), device="cuda", generator=g)
    if n > 1:
        slot = torch.where(torch.rand(n, device="cuda", generator=g) < 0.125, -1, slot)
    cut = torch.sort(torch.randperm(c["S"] - 1, device="cuda", generator=g)[: n - 1] + 1).values
    return slot[torch.bucketize(torch.arange(c["S"], device="cuda"), cut, right=True)].int()


def _rows(c, seed):
    g = _gen(seed, 4)
    x = torch.randn(c["S"], c["I"], device="cuda", generator=g)
    dy = torch.randn(c["S"], c["O"], device="cuda", generator=g) * 0.01
    return x, dy


def _routing(c, seed):
    """Logits [T, E], the K selected experts, row mask, sequence offsets, upstream gradients of the losses.

    The last rows of a batch of several sequences belong to none (padding behind the last one), and one row in
    sixteen is masked."""
    T, E, n = c["T"], c["E"], c["seqs"]
    K = min(c["K"], E)
    g = _gen(seed, 5)
    z = torch.randn(T, E, device="cuda", generator=g) + 0.5 * torch.randn(E, device="cuda", generator=g)
    idx = torch.topk(z, K, dim=1).indices.int()
    mask = (torch.rand(T, device="cuda", generator=g) >= 0.0625).to(torch.uint8)
    used = T if n == 1 else T - T // 32
    cut = torch.sort(torch.randint(0, used + 1, (n - 1,), device="cuda", generator=g)).values
    off = torch.cat((torch.zeros(1, device="cuda", dtype=torch.int64), cut,
                     torch.full((1,), used, device="cuda", dtype=torch.int64))).int()
    return z, idx, mask, off, 0.001 + torch.rand(n, device="cuda", generator=g)


_SESSION = []


def _backend():
    if not _SESSION:
        from colibri_amd.backend import Session
        _SESSION.append(Session(0))
    return _SESSION[0].b


class Held:
    """The tensor and the adapter bank a program keeps, freed together."""

    def __init__(self):
        self.t, self.bank = C.c_void_p(), C.c_void_p()

    def __del__(self):
        if _SESSION:
            if self.bank:
                _SESSION[0].b.hip_lora_free(self.bank)
            if self.t:
                _SESSION[0].b.cuda_tensor_free(self.t)


def _set(b, bank, st):
    """Every adapter of the state into the bank (device pointers, on the backend's stream)."""
    for s, (pa, pb, rank, scale) in enumerate(st["set"]):
        if not b.hip_lora_set_dev(bank, s, pa, pb, rank, scale):
            raise RuntimeError("adapter refused")


def _hold(c, st, q, s):
    """The resident tensor and the bank, and the pointers that the calls take."""
    b, held = _backend(), Held()
    host = s.cpu().numpy()
    torch.cuda.synchronize()   # the upload reads q on the backend's stream
    fp, u8 = C.POINTER(C.c_float), C.POINTER(C.c_uint8)
    mx = c["fmt"] == "mxfp4"
    if not b.hip_tensor_upload_from_device(C.byref(held.t), q.data_ptr(), None if mx else host.ctypes.data_as(fp),
                                           host.ctypes.data_as(u8) if mx else None, 7 if mx else 4, c["I"], c["O"], 0, 32):
        raise RuntimeError("tensor refused")
    st["b"], st["held"] = b, held
    if c["kind"] == "gemm_t":
        return
    if not b.hip_lora_create(C.byref(held.bank), 0, c["I"], c["O"], c["slots"], c["rank"], DTYPES[c["dtype"]][0]):
        raise RuntimeError("adapter bank refused")
    # each adapter as its owner has it: A [rank, I], B [O, rank], contiguous
    st["ab"] = [(st["a"][k, :r].contiguous(), st["bm"][k, :, :r].contiguous()) for k, r in enumerate(_ranks(c))]
    scales = st["scales"].tolist()
    st["set"] = [(a.data_ptr(), bm.data_ptr(), a.shape[0], scales[k]) for k, (a, bm) in enumerate(st["ab"])]
    torch.cuda.synchronize()
    if c["kind"] == "lora":   # a server loads its adapters once
        _set(b, held.bank, st)


def prepare(case, seed):
    c, st = case, {"case": case}
    if c["kind"] == "balance":
        st["z"], st["idx"], st["mask"], st["off"], st["dloss"] = _routing(c, seed)
        n = c["seqs"]
        st["loss"] = torch.zeros(n, device="cuda")
        st["counts"] = torch.zeros(n, c["E"], dtype=torch.int32, device="cuda")
        st["rows"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        st["dz"] = torch.zeros(c["T"], c["E"], device="cuda")
        if own:
            st["b"] = _backend()
        torch.cuda.synchronize()
        return st
    q, s = _weights(c, seed)
    st["x"], st["dy"] = _rows(c, seed)
    st["y"], st["dx"] = torch.zeros_like(st["dy"]), torch.zeros_like(st["x"])
    if c["kind"] != "gemm_t":
        st["a"], st["bm"], st["scales"] = _adapters(c, seed)
        st["slot"] = _slots(c, seed)
    if c["kind"] == "step":
        st["da"] = torch.zeros(c["slots"], c["rank"], c["I"], device="cuda")
        st["db"] = torch.zeros(c["slots"], c["O"], c["rank"], device="cuda")
    if own:
        _hold(c, st, q, s)
    else:
        st["q"], st["s"] = q, s
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------------------------
# one pass: the framework's calls, and the plain form
# ---------------------------------------------------------------------------
def _dequant(c, q, s):
    O, I = c["O"], c["I"]
    n = torch.stack((q & 15, q >> 4), dim=2).reshape(O, -1)[:, :I]
    if c["fmt"] == "mxfp4":
        w = torch.tensor(E2M1, device="cuda")[n.int()]
        s = torch.exp2(s.float() - 127.0)
    else:
        w = n.float() - 8.0
    return w * s.repeat_interleave(32, dim=1)[:, :I]


def _plain_lora(st, grads):
    c = st["case"]
    W = _dequant(c, st["q"], st["s"])
    x, slots, r = st["x"], c["slots"], c["rank"]
    a = st["a"].float().reshape(slots * r, c["I"])
    b = st["bm"].float().permute(0, 2, 1).reshape(slots * r, c["O"])
    # every adapter's product for every row, those of other rows' adapters times zero
    m = (st["slot"][:, None] == torch.arange(slots, device="cuda")[None, :]).float() * st["scales"][None, :]
    m = m.repeat_interleave(r, dim=1)
    h = m * (x @ a.T)
    y = x @ W.T + h @ b
    if not grads:
        return y
    dy = st["dy"]
    dh = m * (dy @ b.T)
    return {"y": y, "dx": dy @ W + dh @ a, "da": (dh.T @ x).reshape(slots, r, c["I"]),
            "db": (h.T @ dy).reshape(slots, r, c["O"]).permute(0, 2, 1).contiguous()}


def _log_score(z, mode):
    if mode == 0:
        return z
    if mode == 3:
        return 0.5 * torch.log(torch.clamp_min(z, 0.0) + torch.log1p(torch.exp(-z.abs())))
    return torch.clamp_max(z, 0.0) - torch.log1p(torch.exp(-z.abs()))


def _plain_balance(st):
    c = st["case"]
    z, mode, n, E = st["z"], c["mode"], c["seqs"], c["E"]
    rows = torch.arange(c["T"], device="cuda")
    seq = torch.bucketize(rows, st["off"][1:].contiguous(), right=True)
    inside = (rows >= st["off"][0]) & (seq < n)
    live = inside & (st["mask"] != 0)
    seq = seq.clamp_max(n - 1)
    u = _log_score(z, mode)
    p = torch.exp(u - u.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    member = (seq[None, :] == torch.arange(n, device="cuda")[:, None]).float() * live[None, :]
    cnt = torch.zeros(n * E, dtype=torch.int32, device="cuda")
    key = (seq[:, None] * E + st["idx"]).reshape(-1)
    cnt.index_add_(0, key, live[:, None].expand_as(st["idx"]).reshape(-1).int())
    counts = cnt.view(n, E)
    nrow = member.sum(1)
    f = E * counts.float() / counts.sum(1, keepdim=True).clamp_min(1).float()
    P = member @ p / nrow.clamp_min(1)[:, None]
    out = {"loss": (f * P).sum(1), "counts": counts, "rows": nrow.int()}
    if c["grad"]:
        w = (st["dloss"] / nrow.clamp_min(1))[:, None] * f
        w = w[seq]
        g = p * (w - (w * p).sum(1, keepdim=True))
        if mode == 3:
            sp = torch.clamp_min(z, 0.0) + torch.log1p(torch.exp(-z.abs()))
            g = g * 0.5 * torch.sigmoid(z) / sp
        elif mode:
            g = g * torch.sigmoid(-z)
        g = g * live[:, None]
        out["dz"] = torch.where(inside[:, None], g, st["dz"])
    return out


def run(state):
    st, c = state, state["case"]
    if not own:
        if c["kind"] == "balance":
            return _plain_balance(st)
        if c["kind"] == "gemm_t":
            return st["dy"] @ _dequant(c, st["q"], st["s"])
        return _plain_lora(st, c["kind"] == "step")
    b = st["b"]
    if c["kind"] == "balance":
        args = (st["mask"].data_ptr(), st["off"].data_ptr(), c["seqs"], c["T"], c["E"])
        ok = b.hip_balance_dev(0, st["z"].data_ptr(), st["idx"].data_ptr(), None, *args, min(c["K"], c["E"]), c["mode"],
                               st["loss"].data_ptr(), st["counts"].data_ptr(), st["rows"].data_ptr())
        out = {"loss": st["loss"], "counts": st["counts"], "rows": st["rows"]}
        if c["grad"]:
            ok = ok and b.hip_balance_grad_dev(0, st["z"].data_ptr(), *args, c["mode"], st["dloss"].data_ptr(),
                                               st["counts"].data_ptr(), st["rows"].data_ptr(), st["dz"].data_ptr())
            out["dz"] = st["dz"]
    elif c["kind"] == "gemm_t":
        ok, out = b.hip_gemm_t_dev(st["held"].t, st["dx"].data_ptr(), st["dy"].data_ptr(), c["S"]), st["dx"]
    else:
        t, bank, x, slot = st["held"].t, st["held"].bank, st["x"].data_ptr(), st["slot"].data_ptr()
        if c["kind"] == "step":
            _set(b, bank, st)
        ok, out = b.hip_lora_gemm_dev(t, bank, st["y"].data_ptr(), x, c["S"], slot), st["y"]
        if c["kind"] == "step":
            ok = ok and b.hip_lora_grad_dev(t, bank, x, st["dy"].data_ptr(), c["S"], slot, st["dx"].data_ptr(),
                                            st["da"].data_ptr(), st["db"].data_ptr())
            out = {k: st[k] for k in ("y", "dx", "da", "db")}
    if not ok:
        raise RuntimeError("the call failed")
    return out


# ---------------------------------------------------------------------------
# the work of one pass, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "balance":
        T, E, n = c["T"], c["E"], c["seqs"]
        by = 4.0 * T * (E + min(c["K"], E)) + T + 4.0 * n * (E + 3)
        fl = 10.0 * T * E
        if c["grad"]:   # the gradient written; its logits are an input already read
            by, fl = by + 4.0 * T * E + 4.0 * n, fl + 10.0 * T * E
        return {"bytes": by, "flops": fl}
    I, O, S = c["I"], c["O"], c["S"]
    wb = O * ((I + 1) // 2) + O * ((I + 31) // 32) * (1 if c["fmt"] == "mxfp4" else 2)
    if c["kind"] == "gemm_t":
        return {"bytes": wb + 4.0 * S * (I + O), "flops": 2.0 * S * I * O}
    ranks = _ranks(c)
    size = 4 if c["dtype"] == "f32" else 2
    used = sum(ranks[: min(c["slots"], c["requests"])])
    mean = sum(ranks) / len(ranks)
    by = wb + used * size * (I + O) + 4.0 * S * (I + O + 1)
    fl = 2.0 * S * I * O + 2.0 * S * mean * (I + O)
    if c["kind"] == "step":   # dy read, dx, dA and dB written; four more products of the rank's size
        by += 4.0 * S * (I + O) + 4.0 * c["slots"] * c["rank"] * (I + O)
        fl += 2.0 * S * I * O + 4.0 * S * mean * (I + O)
    return {"bytes": by, "flops": fl}


def _w64(c, seed):
    q, s = _weights(c, seed)
    w = torch.empty(c["O"], 2 * q.shape[1], dtype=torch.float64, device="cuda")
    if c["fmt"] == "mxfp4":
        table = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = table[(q & 15).long()], table[(q >> 4).long()]
        scale = torch.ldexp(torch.ones((), dtype=torch.float64, device="cuda"), s.int() - 127)
    else:
        w[:, 0::2], w[:, 1::2] = (q & 15).double() - 8.0, (q >> 4).double() - 8.0
        scale = s.double()
    w = w[:, : c["I"]].contiguous()
    return w * scale[:, torch.arange(c["I"], device="cuda") // 32]


def _exact_balance(c, seed):
    z, idx, mask, off, dloss = (v.cpu() for v in _routing(c, seed))
    z, E, n = z.double(), c["E"], c["seqs"]
    if c["mode"] == 0:
        p, up = torch.softmax(z, 1), torch.ones_like(z)
    elif c["mode"] == 3:
        s = torch.sqrt(torch.nn.functional.softplus(z, threshold=700.0))
        p, up = s / s.sum(1, keepdim=True), torch.sigmoid(z) / (2.0 * s * s)
    else:
        s = torch.sigmoid(z)
        p, up = s / s.sum(1, keepdim=True), 1.0 - s
    loss, counts = torch.zeros(n, dtype=torch.float64), torch.zeros(n, E, dtype=torch.int32)
    rows, dz = torch.zeros(n, dtype=torch.int32), torch.zeros_like(z)
    for i in range(n):
        at = torch.arange(int(off[i]), int(off[i + 1]))
        at = at[mask[at] != 0]
        if not len(at):
            continue
        rows[i] = len(at)
        counts[i] = torch.bincount(idx[at].reshape(-1).long(), minlength=E).int()
        f = counts[i].double() * E / counts[i].sum()
        pr = p[at]
        loss[i] = (f * pr.mean(0)).sum()
        w = float(dloss[i]) / len(at) * f
        dz[at] = pr * (w - (pr @ w)[:, None]) * up[at]
    out = {"loss": loss, "counts": counts, "rows": rows}
    if c["grad"]:
        out["dz"] = dz
    return out


def exact(case, seed):
    c = case
    if c["kind"] == "balance":
        return _exact_balance(c, seed)
    w = _w64(c, seed)
    x, dy = (v.double() for v in _rows(c, seed))
    if c["kind"] == "gemm_t":
        return dy @ w
    a, b, scales = (v.double() for v in _adapters(c, seed))
    slot = _slots(c, seed)
    y, dx = x @ w.T, dy @ w
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for k in range(c["slots"]):
        at = torch.nonzero(slot == k)[:, 0]
        h, dh = scales[k] * (x[at] @ a[k].T), scales[k] * (dy[at] @ b[k])
        y[at] += h @ b[k].T
        dx[at] += dh @ a[k]
        da[k], db[k] = dh.T @ x[at], dy[at].T @ h
    return {"y": y, "dx": dx, "da": da, "db": db} if c["kind"] == "step" else y
