"""Cases of the operators that train LoRA adapters on frozen int4 weights.

  act8           a layer's input kept for its backward pass in 8 bits (int8 codes, one power-of-two step per 32
                 values of a row) and read back;
  lora_act8      the adapter's gradients dA = s X^T (dY B^T), dB = s (X A)^T dY from X kept in 8 bits;
  input_grad     dX = dY W^T + s (dY B^T) A^T through the frozen int4 weights W [k, n] and the adapter;
  loss           softmax cross entropy of X W over a vocabulary of n columns, and its gradient in X.

``own`` false: plain torch operations in 32 bits.  ``own`` true: the calls of the framework's Python binding.
Weights are in the framework's layout: packed [n, k/8] words (8 nibbles, lowest k first), scales [n, k/32].
"""
import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
IGNORED = -100  # target of a row that takes no part in the loss


def listed():
    return [
        # one token's hidden state of a 4096-wide layer: latency
        dict(name="act8 one row", op="act8", m=1, k=4096, dtype="f32"),
        # a 2048-token batch at the input of the 4096-wide projections
        dict(name="act8 2048x4096 f32", op="act8", m=2048, k=4096, dtype="f32"),
        # the wide side of a 7B MLP, bf16 activations, an odd row count
        dict(name="act8 4095x11008 bf16", op="act8", m=4095, k=11008, dtype="bf16"),
        # the smallest layer: 64 -> 256, rank 4
        dict(name="lora_act8 64x256", op="lora_act8", m=128, k=64, n=256, rank=4, dtype="f32"),
        # a 512-token step of a square 4096 layer with rank 16, fp32 gradients
        dict(name="lora_act8 512 f32", op="lora_act8", m=512, k=4096, n=4096, rank=16, dtype="f32"),
        # a 4096-token step of the MLP up-projection, bf16 gradients
        dict(name="lora_act8 4096 bf16", op="lora_act8", m=4096, k=4096, n=11008, rank=16, dtype="bf16"),
        # a handful of rows (the last, short batch) through a square layer
        dict(name="input_grad 7 rows", op="input_grad", m=7, k=4096, n=4096, rank=16, dtype="f32"),
        # ragged rows and columns, no adapter on this layer, fp32
        dict(name="input_grad 515 f32", op="input_grad", m=515, k=2080, n=4099, rank=0, dtype="f32"),
        # the MLP up-projection's input gradient of a 2048-token batch with the adapter
        dict(name="input_grad 2048 bf16", op="input_grad", m=2048, k=4096, n=11008, rank=16, dtype="bf16"),
        # the loss of a few tokens alone (scoring), an odd vocabulary
        dict(name="loss 5 rows", op="loss", m=5, k=1024, n=32003, dtype="f32", grad=False),
        # loss and gradient of a batch in fp32, an odd vocabulary
        dict(name="loss 1000 f32", op="loss", m=1000, k=2048, n=50001, dtype="f32", grad=True),
        # loss and gradient of a 4096-token batch over a large vocabulary in bf16
        dict(name="loss 4096 bf16", op="loss", m=4096, k=4096, n=65536, dtype="bf16", grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["act8", "lora_act8", "input_grad", "loss"])
    c = dict(op=op, m=_log(rng, 1, 4096), k=32 * _log(rng, 2, 344 if op == "act8" else 192), dtype=rng.choice(["f32", "bf16"]))
    if op in ("lora_act8", "input_grad"):
        c["n"] = rng.choice([1, 8]) * _log(rng, 33, 1400)
        c["rank"] = rng.choice([1, 4, 8, 16, 16, 33, 64]) if op == "lora_act8" else rng.choice([0, 0, 5, 16, 64])
    if op == "loss":
        c["n"] = _log(rng, 257, 65536)
        c["grad"] = rng.random() < 0.75
        while c["m"] * c["k"] * c["n"] > 4096 * 4096 * 65536:
            c["m"] = (c["m"] + 1) // 2
    return c


# ------------------------------------------------------------------ inputs --
def _package():
    """spaceslug-main_b200/ as the module ``spaceslug_b200`` (its folder's name is no module name)."""
    if "spaceslug_b200" not in sys.modules:
        root = Path.cwd() / "spaceslug-main_b200"
        spec = importlib.util.spec_from_file_location("spaceslug_b200", root / "__init__.py",
                                                      submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["spaceslug_b200"] = mod
        spec.loader.exec_module(mod)
    from spaceslug_b200 import backend
    return backend


class _Handle:
    """A weight handle that frees its device memory with the state that holds it."""

    def __init__(self, s):
        self.session = _package().BackendSession()
        n, k = s["scales"].shape[0], s["scales"].shape[1] * 32
        self.w = self.session.weights(s["packed"].cpu().numpy().view(np.uint32), s["scales"].cpu().numpy(), k, n)
        if s.get("a") is not None:
            self.w.set_lora(s["a"].cpu().numpy(), s["b"].cpu().numpy(), s["alpha"])

    def __del__(self):
        torch.cuda.synchronize()
        self.w.close()


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m, k, dt = c["m"], c["k"], DT[c["dtype"]]
    n, r = c.get("n", 0), c.get("rank", 0)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = dict(op=c["op"], dtype=c["dtype"], grad=c.get("grad", True))
    if c["op"] != "act8":
        s["packed"] = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=g, device="cuda", dtype=torch.int32)
        s["scales"] = 0.002 + 0.008 * torch.rand((n, k // 32), generator=g, device="cuda")
    if r:
        s["a"], s["b"], s["alpha"] = 0.02 * normal(k, r), 0.02 * normal(r, n), 2.0 * r
    # hidden states: normal, with a few channels that are an order larger, as behind a norm's learned weights
    x = normal(m, k) * (1.0 + 9.0 * (torch.rand((k,), generator=g, device="cuda") < 0.005))
    if c["op"] == "act8":
        s["x"] = x.to(dt)
    if c["op"] == "lora_act8":
        s["codes"], s["exps"] = _pack(x)
    if c["op"] in ("lora_act8", "input_grad"):
        s["dy"] = (normal(m, n) * (0.1 * torch.rand((m, 1), generator=g, device="cuda"))).to(dt)
    if c["op"] == "loss":
        # one row in ten is ignored; the others lean towards their target as a trained model's do
        t = torch.randint(0, n, (m,), generator=g, device="cuda")
        w = _dequant(s["packed"][t], s["scales"][t], torch.float32)
        lean = 10.0 * torch.rand((m, 1), generator=g, device="cuda") / w.square().sum(1, keepdim=True)
        s["x"] = (normal(m, k) * 0.5 + lean * w).to(dt)
        s["targets"] = torch.where(torch.rand((m,), generator=g, device="cuda") < 0.1, IGNORED, t)
        s["row_scale"] = torch.full((m,), 1.0 / m, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["session"] = _package().BackendSession()
        if "packed" in s:
            s["handle"] = _Handle(s)
    return s


# -------------------------------------------------------------- plain form --
def _dequant(packed, scales, dtype):
    """[n, k] weights of packed [n, k/8] and scales [n, k/32]."""
    n, words = packed.shape
    shifts = torch.arange(0, 32, 4, device=packed.device, dtype=torch.int32)
    v = (((packed.unsqueeze(-1) >> shifts) & 15) ^ 8) - 8
    return (v.view(n, words // 4, 32).to(dtype) * scales.to(dtype).unsqueeze(-1)).view(n, words * 8)


def _pack(x):
    """8-bit codes [m, k] and step exponents (biased by 127) [m, k/32]: the step of a group is the smallest power of
    two of which its largest value takes at most 127 steps."""
    m, k = x.shape
    grp = x.float().view(m, k // 32, 32)
    f, e = torch.frexp(grp.abs().amax(-1))  # amax = f 2^e, f in [0.5, 1)
    e = (e.to(torch.int32) - 7 + (f > 127.0 / 128.0).to(torch.int32)).clamp(min=-126)
    codes = torch.round(torch.ldexp(grp, -e.unsqueeze(-1))).to(torch.int8).view(m, k)
    return codes, (e + 127).to(torch.uint8)


def _unpack(codes, exps):
    m, k = codes.shape
    step = torch.ldexp(torch.ones_like(exps, dtype=torch.float32), exps.to(torch.int32) - 127)
    return (codes.view(m, k // 32, 32).float() * step.unsqueeze(-1)).view(m, k)


def _plain(s):
    dt = DT[s["dtype"]]
    if s["op"] == "act8":
        return _unpack(*_pack(s["x"])).to(dt)
    if s["op"] == "lora_act8":
        x, dy, scale = _unpack(s["codes"], s["exps"]), s["dy"].float(), s["alpha"] / s["a"].shape[1]
        return dict(da=scale * (x.T @ (dy @ s["b"].T)), db=scale * ((x @ s["a"]).T @ dy))
    w = _dequant(s["packed"], s["scales"], torch.float32)
    if s["op"] == "input_grad":
        dy = s["dy"].float()
        dx = dy @ w
        if "a" in s:
            dx = dx + (s["alpha"] / s["a"].shape[1]) * ((dy @ s["b"].T) @ s["a"].T)
        return dx.to(dt)
    z = s["x"].float() @ w.T
    used = s["targets"] >= 0
    t = s["targets"].clamp(min=0)
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    loss = torch.where(used, lse - z.gather(1, t.unsqueeze(1)).squeeze(1), 0.0)
    if not s["grad"]:
        return dict(loss=loss, lse=lse)
    p = p / total
    rows = torch.arange(p.shape[0], device=p.device)
    p[rows, t] -= 1.0
    dx = (p * torch.where(used, s["row_scale"], 0.0).unsqueeze(1)) @ w
    return dict(loss=loss, lse=lse, dx=dx.to(dt))


# ------------------------------------------------------- the framework's calls --
def _own(s):
    st = torch.cuda.current_stream().cuda_stream
    ses, d = s["session"], s["dtype"]
    if s["op"] == "act8":
        x = s["x"]
        m, k = x.shape
        codes = torch.empty((m, k), dtype=torch.int8, device=x.device)
        exps = torch.empty((m, k // 32), dtype=torch.uint8, device=x.device)
        out = torch.empty_like(x)
        ses.act8_pack_device(x.data_ptr(), codes.data_ptr(), exps.data_ptr(), m, k, dtype=d, stream=st)
        ses.act8_unpack_device(codes.data_ptr(), exps.data_ptr(), out.data_ptr(), m, k, dtype=d, stream=st)
        return out
    w = s["handle"].w
    if s["op"] == "lora_act8":
        m, r = s["dy"].shape[0], s["a"].shape[1]
        da = torch.empty((w.k, r), device=s["dy"].device)
        db = torch.empty((r, w.n), device=s["dy"].device)
        w.lora_backward_act8(s["codes"].data_ptr(), s["exps"].data_ptr(), s["dy"].data_ptr(), m, dtype=d,
                             da=da.data_ptr(), db=db.data_ptr(), stream=st)
        return dict(da=da, db=db)
    if s["op"] == "input_grad":
        m = s["dy"].shape[0]
        dx = torch.empty((m, w.k), dtype=DT[d], device=s["dy"].device)
        w.input_gradient(s["dy"].data_ptr(), dx.data_ptr(), m, dtype=d, stream=st)
        return dx
    x = s["x"]
    m = x.shape[0]
    loss, lse = torch.empty((m,), device=x.device), torch.empty((m,), device=x.device)
    dx = torch.empty_like(x) if s["grad"] else None
    w.cross_entropy(x.data_ptr(), s["targets"].data_ptr(), loss.data_ptr(), m, lse=lse.data_ptr(),
                    dx=dx.data_ptr() if s["grad"] else 0, row_scale=s["row_scale"].data_ptr() if s["grad"] else 0,
                    dtype=d, stream=st)
    return dict(loss=loss, lse=lse, dx=dx) if s["grad"] else dict(loss=loss, lse=lse)


def run(state):
    return _own(state) if own else _plain(state)


# -------------------------------------------------------------------- work --
def work(case):
    m, k, n, r = case["m"], case["k"], case.get("n", 0), case.get("rank", 0)
    size = 4 if case["dtype"] == "f32" else 2
    kept = m * k + m * k // 32  # codes and exponents
    weights = n * k // 2 + n * (k // 32) * 4
    adapter = 4 * r * (k + n)
    if case["op"] == "act8":  # x read, kept written; kept read, x written
        return dict(bytes=2 * (m * k * size + kept), flops=4 * m * k)
    if case["op"] == "lora_act8":
        return dict(bytes=kept + m * n * size + 2 * adapter, flops=4 * m * r * (k + n))
    if case["op"] == "input_grad":
        return dict(bytes=weights + adapter + m * (n + k) * size, flops=2 * m * n * k + 2 * m * r * (k + n))
    if not case["grad"]:
        return dict(bytes=weights + m * k * size + 16 * m, flops=2 * m * n * k)
    return dict(bytes=weights + 2 * m * k * size + 20 * m, flops=4 * m * n * k)


# ------------------------------------------------------------------- exact --
def _w64(s):
    """W as [k, n] in 64 bits, nibble by nibble from the bytes of the layout: byte n (k/2) + k/2, even k low."""
    by = s["packed"].view(torch.uint8).to(torch.int64)
    v = torch.stack((by % 16, by // 16), dim=-1).flatten(1)
    v = torch.where(v > 7, v - 16, v).double()
    return (v * s["scales"].double().repeat_interleave(32, dim=1)).T


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "act8":
        x = s["x"].double().unflatten(1, (-1, 32))
        top = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top / 127.0))  # smallest e with top <= 127 2^e, put right where log2 rounds
        e = e + (top > 127.0 * torch.exp2(e)).double()
        e = e - (top <= 127.0 * torch.exp2(e - 1.0)).double()
        e = torch.where(top > 0, e, -126.0).clamp(min=-126.0)
        return (torch.round(x / torch.exp2(e)) * torch.exp2(e)).flatten(1)
    if case["op"] == "lora_act8":
        x = s["codes"].double() * torch.exp2(s["exps"].double() - 127.0).repeat_interleave(32, dim=1)
        dy, a, b = s["dy"].double(), s["a"].double(), s["b"].double()
        scale = s["alpha"] / case["rank"]
        return dict(da=scale * torch.einsum("mk,mr->kr", x, torch.einsum("mn,rn->mr", dy, b)),
                    db=scale * torch.einsum("mr,mn->rn", torch.einsum("mk,kr->mr", x, a), dy))
    w = _w64(s)
    if case["op"] == "input_grad":
        dy = s["dy"].double()
        if case["rank"]:
            w = w + (s["alpha"] / case["rank"]) * (s["a"].double() @ s["b"].double())
        return torch.einsum("mn,kn->mk", dy, w)
    z = torch.einsum("mk,kn->mn", s["x"].double(), w)
    lse = torch.logsumexp(z, dim=1)
    hot = torch.zeros_like(z)
    used = (s["targets"] != IGNORED).double()
    hot[torch.arange(z.shape[0], device=z.device), torch.where(used > 0, s["targets"], 0)] = used
    loss = lse * used - (hot * torch.where(hot > 0, z, 0.0)).sum(1)
    if not case["grad"]:
        return dict(loss=loss, lse=lse)
    prob = torch.exp(z - lse.unsqueeze(1)) * used.unsqueeze(1)
    return dict(loss=loss, lse=lse, dx=torch.einsum("mn,kn->mk", (prob - hot) * s["row_scale"].double().unsqueeze(1), w))
