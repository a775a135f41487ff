"""One 8-bit expert layer, forwards and backwards, on the library's operators.

A mixture-of-experts layer whose weights are e4m3 with a scale for each 128 x
128 block: the router's balance over packed documents, the experts' gate/up
and down products over rows grouped by expert, and both gradients of the down
product -- with regard to its input (through the weight laid out by columns)
and to each expert's weight (both operands quantised along the tokens).

torch only holds the buffers and does the steps that the library has no
operator for (routing by top-k, the gate, the weighted sum).

    python examples/fp8_expert_layer.py [--tokens 4096] [--experts 128] ...
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from textsift_b200 import abi  # noqa: E402

BLOCK = 128
DTYPES = {torch.float16: abi.TS_DTYPE_F16, torch.bfloat16: abi.TS_DTYPE_BF16, torch.float32: abi.TS_DTYPE_F32}


def _up(n: int, m: int) -> int:
    return -(-n // m) * m


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


class Operand:
    """Rows of 8-bit codes [R, pitch] and their scales [blocks, R rounded up]."""

    def __init__(self, rows: int, cols: int):
        self.rows, self.cols = rows, cols
        self.codes = torch.empty(rows, _up(cols, 16), dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(_up(cols, BLOCK) // BLOCK, _up(rows, 4), device="cuda")


def quantise(x: torch.Tensor, by_columns: bool = False) -> Operand:
    rows, cols = x.shape
    o = Operand(cols, rows) if by_columns else Operand(rows, cols)
    abi.check(abi.lib().ts_cuda_op_quant_fp8(
        x.data_ptr(), DTYPES[x.dtype], x.stride(0), rows, cols, int(by_columns), o.codes.data_ptr(), o.codes.stride(0),
        o.scales.data_ptr(), o.scales.stride(0), _stream()))
    return o


class Weight:
    """Expert weights [E, N, K] as codes and block scales, and the same by columns for the gradient of their input."""

    def __init__(self, w: torch.Tensor):
        e, n, k = w.shape
        self.e, self.n, self.k = e, n, k
        full = torch.zeros(e, _up(n, BLOCK), _up(k, BLOCK), device="cuda")
        full[:, :n, :k] = w
        v = full.view(e, full.shape[1] // BLOCK, BLOCK, full.shape[2] // BLOCK, BLOCK)
        # the format's roundings: the scale is the largest magnitude times f32(1/448), the codes are those of v times
        # the scale's f32 reciprocal
        self.scales = (v.abs().amax((2, 4)) * (1.0 / 448.0)).clamp_min(2.0 ** -100).contiguous()
        q = (v * (1.0 / self.scales)[:, :, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        self.codes = torch.zeros(e, n, _up(k, 16), dtype=torch.uint8, device="cuda")
        self.codes[:, :, :k] = q.view(e, full.shape[1], full.shape[2])[:, :n, :k].view(torch.uint8)
        self.codes_t = torch.zeros(e, k, _up(n, 16), dtype=torch.uint8, device="cuda")
        self.scales_t = torch.empty(e, self.scales.shape[2], self.scales.shape[1], device="cuda")
        abi.check(abi.lib().ts_cuda_op_transpose_fp8(
            self.codes.data_ptr(), self.codes.stride(1), self.scales.data_ptr(), e, n, k, self.codes_t.data_ptr(),
            self.codes_t.stride(1), self.scales_t.data_ptr(), _stream()))

    def value(self) -> torch.Tensor:
        """The f32 weight that the codes stand for."""
        s = self.scales.repeat_interleave(BLOCK, 1)[:, :self.n].repeat_interleave(BLOCK, 2)[:, :, :self.k]
        return self.codes.view(torch.float8_e4m3fn)[:, :, :self.k].float() * s

    def _product(self, a: Operand, codes, scales, n: int, k: int, seg: torch.Tensor, dtype) -> torch.Tensor:
        out = torch.empty(a.rows, n, dtype=dtype, device="cuda")
        abi.check(abi.lib().ts_cuda_op_matmul_fp8(
            a.codes.data_ptr(), a.codes.stride(0), a.scales.data_ptr(), a.scales.stride(0), codes.data_ptr(),
            codes.stride(1), scales.data_ptr(), 0, BLOCK, None, seg.data_ptr(), self.e, out.data_ptr(), DTYPES[dtype], n,
            0, a.rows, n, k, _stream()))
        return out

    def forward(self, a: Operand, seg: torch.Tensor, dtype=torch.float16) -> torch.Tensor:
        return self._product(a, self.codes, self.scales, self.n, self.k, seg, dtype)

    def grad_input(self, dy: Operand, seg: torch.Tensor, dtype=torch.float16) -> torch.Tensor:
        return self._product(dy, self.codes_t, self.scales_t, self.k, self.n, seg, dtype)


def grad_weight(dy: torch.Tensor, x: torch.Tensor, dw: torch.Tensor) -> None:
    """dw [N, K] f32 += dy [T, N] transposed times x [T, K]."""
    a, b = quantise(dy, by_columns=True), quantise(x, by_columns=True)
    abi.check(abi.lib().ts_cuda_op_matmul_fp8(
        a.codes.data_ptr(), a.codes.stride(0), a.scales.data_ptr(), a.scales.stride(0), b.codes.data_ptr(),
        b.codes.stride(0), b.scales.data_ptr(), b.scales.stride(0), 1, None, None, 1, dw.data_ptr(), abi.TS_DTYPE_F32,
        dw.stride(0), 1, dw.shape[0], dw.shape[1], dy.shape[0], _stream()))


def balance(logits: torch.Tensor, idx: torch.Tensor, seq: torch.Tensor, alpha: float):
    """(counts [S, E], prob [S, E], loss, gradient of the logits) over the documents that seq bounds."""
    t, e = logits.shape
    s, lib = seq.numel() - 1, abi.lib()
    counts = torch.empty(s, e, dtype=torch.int32, device="cuda")
    prob, loss = torch.empty(s, e, device="cuda"), torch.empty(1, device="cuda")
    grad = torch.empty_like(logits)
    work = torch.empty(lib.ts_cuda_router_balance_work(s, e), dtype=torch.uint8, device="cuda")
    abi.check(lib.ts_cuda_op_router_balance(
        logits.data_ptr(), DTYPES[logits.dtype], logits.stride(0), idx.data_ptr(), None, seq.data_ptr(), s, t, e,
        idx.shape[1], alpha, 1.0, counts.data_ptr(), prob.data_ptr(), loss.data_ptr(), grad.data_ptr(), grad.stride(0),
        work.data_ptr(), work.numel(), _stream()))
    return counts, prob, loss, grad


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    gate, up = gu[:, 0::2].float().clamp(max=7.0), gu[:, 1::2].float().clamp(-7.0, 7.0)
    return ((up + 1.0) * gate * torch.sigmoid(1.702 * gate)).half()


def step(x: torch.Tensor, router: torch.Tensor, gate_up: Weight, down: Weight, seq: torch.Tensor, k: int,
         dy: torch.Tensor):
    """One forward of the layer and the gradients of its down product for dy [T, D]."""
    logits = x.float() @ router.float().t()
    top = logits.topk(k, dim=1)
    idx, weight = top.indices.to(torch.int32), torch.softmax(top.values, 1)
    counts, prob, loss, dlogits = balance(logits, idx, seq, 0.01)
    # rows grouped by expert; the segments are the sums of the balance's counts
    seg = torch.zeros(gate_up.e + 1, dtype=torch.int32, device="cuda")
    seg[1:] = counts.sum(0).cumsum(0)
    order = idx.flatten().argsort(stable=True)
    token = order // k
    g = swiglu(gate_up.forward(quantise(x[token]), seg))
    routes = down.forward(quantise(g), seg)
    y = torch.zeros(x.shape, device="cuda").index_add_(0, token, routes.float() * weight.flatten()[order, None])
    droutes = (dy[token].float() * weight.flatten()[order, None]).half()
    dg = down.grad_input(quantise(droutes), seg)
    dw = torch.zeros(down.e, down.n, down.k, device="cuda")
    ends = seg.tolist()
    for e in range(down.e):
        if ends[e + 1] > ends[e]:
            grad_weight(droutes[ends[e]:ends[e + 1]], g[ends[e]:ends[e + 1]], dw[e])
    return {"y": y, "routes": routes, "weight": weight.flatten()[order], "loss": loss, "counts": counts, "prob": prob, "dlogits": dlogits, "seg": seg, "order": order, "g": g,
            "dg": dg, "dw": dw, "droutes": droutes}


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--experts", type=int, default=128)
    ap.add_argument("--hidden", type=int, default=640)
    ap.add_argument("--k", type=int, default=4)
    ap.add_argument("--documents", type=int, default=5)
    a = ap.parse_args(argv)
    gen = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    d = a.hidden
    x, dy = rand(a.tokens, d).half(), rand(a.tokens, d).half()
    router = rand(a.experts, d) / d ** 0.5
    gate_up, down = Weight(rand(a.experts, 2 * d, d) / d ** 0.5), Weight(rand(a.experts, d, d) / d ** 0.5)
    seq = torch.linspace(0, a.tokens, a.documents + 1, device="cuda").int()
    out = step(x, router, gate_up, down, seq, a.k, dy)
    abi.check(abi.lib().ts_cuda_op_check(_stream()))
    # the same in f32 on the weights that the codes stand for
    seg, token = out["seg"].tolist(), out["order"] // a.k
    wu, wd = gate_up.value(), down.value()
    err = {"forward": 0.0, "down product": 0.0, "input gradient": 0.0, "weight gradient": 0.0}
    y = torch.zeros(x.shape, device="cuda")
    for e in range(a.experts):
        r = slice(seg[e], seg[e + 1])
        if seg[e] == seg[e + 1]:
            continue
        g = swiglu((x[token[r]].float() @ wu[e].t()).half())
        routes = out["g"][r].float() @ wd[e].t()
        y.index_add_(0, token[r], routes * out["weight"][r, None])
        pairs = {"forward": (out["g"][r].float(), g.float()),
                 "down product": (out["routes"][r].float(), routes),
                 "input gradient": (out["dg"][r].float(), out["droutes"][r].float() @ wd[e]),
                 "weight gradient": (out["dw"][e], out["droutes"][r].float().t() @ out["g"][r].float())}
        for name, (got, want) in pairs.items():
            err[name] = max(err[name], float((got - want).norm() / want.norm()))
    err["output"] = float((out["y"] - y).norm() / y.norm())
    print(f"{a.tokens} tokens, {a.experts} experts: balance loss {float(out['loss']):.6f}, routes per expert "
          f"{int(out['counts'].sum(0).min())}..{int(out['counts'].sum(0).max())}; largest errors against f32: "
          + ", ".join(f"{n} {v:.3f}" for n, v in err.items()))
    return {**out, "errors": err}


if __name__ == "__main__":
    main()
