"""Runs the paged attention's tensor-core entries in the CPU emulator (:mod:`tests.tcemu`), with the packed
16-bit subtraction its byte conversion uses; test infrastructure only."""
from __future__ import annotations

import numpy as np

from emmy_ptx_b200.compiler import compile_graph
from emmy_ptx_b200.data import from_numpy_storage, to_numpy_storage
from emmy_ptx_b200.ir import Graph
from tests.ptxemu import Memory
from tests.tcemu import TcEmulator, _halves_to_float
from oracle.interp import f32_to_bf16_bits


class PagedEmulator(TcEmulator):
    @staticmethod
    def _decode(x):
        if not x.label and x.op.startswith(("sub.rn.bf16x2", "sub.rn.f16x2")):
            return (7,)
        return TcEmulator._decode(x)

    def _extra(self, th, x, op, ops, regs, val, addr, smem, mem):
        if op.startswith(("sub.rn.bf16x2", "sub.rn.f16x2")):
            bf = "bf16" in op
            a, b = (np.array([val(o) & 0xFFFF, (val(o) >> 16) & 0xFFFF], np.uint16) for o in ops[1:3])
            r = (_halves_to_float(a, int(bf)) - _halves_to_float(b, int(bf))).astype(np.float32)
            bits = f32_to_bf16_bits(r) if bf else r.astype(np.float16).view(np.uint16)
            regs[ops[0]] = int(bits[0]) | int(bits[1]) << 16
            return "cont"
        return super()._extra(th, x, op, ops, regs, val, addr, smem, mem)


def run(p, t, opts=None, defer=False, mod=None):
    """(outputs, error word, module): the problem compiled with ``opts`` and run on CPU tensors ``t``; scratch starts
    as NaN, so a part that is read without having been written shows."""
    mod = mod or compile_graph(Graph.from_dict(p.graph), p.meta(), opts or {})
    mem = Memory()
    addr = {a.name: mem.alloc(to_numpy_storage(t[a.name])) for a in p.args}
    for rec in mod.kernels:
        for spec in rec.get("scratch", []):
            n = int(np.prod(spec["shape"]))
            addr.setdefault(spec["name"], mem.alloc(np.full(n, np.nan, np.float32)))
    err = mem.alloc(np.zeros(16, np.uint8))
    for rec in mod.kernels:
        tm = {f"p_{s['name']}": (addr[s["tensor"]], s) for s in rec.get("tmaps", [])}
        emu = PagedEmulator(mod.ptx, rec["entry"], tm, defer=defer)
        plain = [q for q in emu.params if not q.startswith("p_tm") and q != "p_err"]
        args = dict(zip(plain, [addr[n] for n in rec["params"]]))
        args.update(emu.tmap_args())
        args["p_err"] = err
        emu.run(rec["grid"][0], rec["block"][0], args, mem, rec.get("dyn_smem", 0))
    out = {}
    for a in p.outputs:
        host = to_numpy_storage(t[a.name])
        out[a.name] = from_numpy_storage(mem.array(addr[a.name], host.dtype, (-1,)).copy(), a.dtype).reshape(a.shape)
    return out, int(mem.array(err, np.int32, (4,))[0]), mod
