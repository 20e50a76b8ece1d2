"""Runs the paged attention's tensor-core entries in the CPU emulator (:mod:`tests.tcemu`), with what they
use beyond it: packed 16-bit subtractions, warp matrix products and plain bulk copies; test infrastructure only."""
from __future__ import annotations

import numpy as np

from emmy_ptx_b200.compiler import compile_graph
from emmy_ptx_b200.data import from_numpy_storage, to_numpy_storage
from emmy_ptx_b200.ir import Graph
from tests.ptxemu import Memory
from tests.tcemu import TcEmulator, _halves_to_float
from oracle.interp import f32_to_bf16_bits


_OWN = ("popc.b32", "sub.rn.bf16x2", "sub.rn.f16x2", "mma.sync", "cp.async.bulk.shared")


class PagedEmulator(TcEmulator):
    """``mma.sync`` m16n8k16 is a warp's collective; plain bulk copies complete like TMA boxes."""

    @staticmethod
    def _decode(x):
        if not x.label and x.op.startswith(_OWN):
            return (7,)                                     # straight to _extra
        return TcEmulator._decode(x)

    def _tma_write(self, dst, tm, cs, mb, smem, mem):
        if isinstance(tm, tuple):
            smem[dst:dst + tm[2]] = mem.load(tm[1], tm[2])
            return self._complete_tx(mb, tm[2])
        return super()._tma_write(dst, tm, cs, mb, smem, mem)

    def _collective(self, members, args):
        if not members[0].coll[0].startswith("mma.sync"):
            return super()._collective(members, args)
        ins = self.ins[members[0].pc]
        groups = [[r.strip() for r in o.strip().strip("{}").split(",")] for o in ins.ops]
        D, A, B, C = groups
        bf = int("bf16" in ins.op)
        lanes = sorted(members, key=lambda t: t.lane)
        halves = lambda v: _halves_to_float(np.array([v & 0xFFFF, v >> 16 & 0xFFFF], np.uint16), bf)
        a, b, c = np.zeros((16, 16)), np.zeros((16, 8)), np.zeros((16, 8))
        for t in lanes:
            g, q = t.lane >> 2, t.lane & 3
            for r in range(4):
                a[g + 8 * (r & 1), 2 * q + 8 * (r >> 1):2 * q + 8 * (r >> 1) + 2] = halves(t.regs[A[r]])
                c[g + 8 * (r >> 1), 2 * q + (r & 1)] = np.uint32(t.regs[C[r]]).view(np.float32)
            for r in range(2):
                b[2 * q + 8 * r:2 * q + 8 * r + 2, g] = halves(t.regs[B[r]])
        with np.errstate(all="ignore"):
            d = (a @ b + c).astype(np.float32)
        for t in lanes:
            g, q = t.lane >> 2, t.lane & 3
            for r in range(4):
                t.regs[D[r]] = int(d[g + 8 * (r >> 1), 2 * q + (r & 1)].view(np.uint32))

    def _extra(self, th, x, op, ops, regs, val, addr, smem, mem):
        if op.startswith("popc.b32"):
            regs[ops[0]] = bin(val(ops[1]) & 0xFFFFFFFF).count("1")
            return "cont"
        if op.startswith("mma.sync"):
            th.pc -= 1
            th.state, th.coll = "coll", (op, 0xFFFFFFFF)
            return "block"
        if op.startswith("cp.async.bulk.shared::cluster.global"):
            dst, src, n, mb = addr(ops[0]) & 0xFFFFFFFF, addr(ops[1]), val(ops[2]), addr(ops[3]) & 0xFFFFFFFF
            assert dst % 16 == 0 and src % 16 == 0 and n % 16 == 0 and dst + n <= len(smem), (dst, src, n)
            if self.defer:
                self.queue_tma.append((dst, ("bulk", src, n), None, mb, mem))
            else:
                smem[dst:dst + n] = mem.load(src, n)
                self._complete_tx(mb, n)
            return "cont"
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
