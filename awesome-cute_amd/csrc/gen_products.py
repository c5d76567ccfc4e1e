#!/usr/bin/env python3
"""Writes the main loops of the big tiles of the feed-forward products (ff_big.hip) as inline
assembly statements with fixed registers: for fp16 and bfloat16, for tiles of 32 rb rows (rb =
5 ... 8) x 256 columns, and for operands by rows of the summed dimension's length or turned
over, as rows along the output ("TurnB": B so, "TurnBoth": A too).

A workgroup has four waves, one per SIMD, two by two, each with an accumulator of 16 rb x 128 in
AGPRs; why assembly, and why that shape, says gen_dense.py, whose schedule this is with the
number of row blocks, the reads per operand and the requests as parameters.

A step is 8 rb MFMAs over 32 k-values: row blocks i = 0 ... rb - 1 of 16 rows, operands o = 0 ... 7
of 16 columns.  A slab, 64 k-values, is two steps.  LDS holds three slabs of B and two of A (three of 160 rows): of the two it
is B, a model's weights, that comes from memory, and a load's way from there is longer than a
slab's MFMAs (two and two: 2048 x 10752 x 4096, B turned over, 136 us with operands in the last-level
cache and 175 from memory).  A operands are read
`ahead` row blocks ahead, each row block into registers of its own; the eight B operands of the
next step go into the other of two buffers:

  inner step (the next step is in the same slab)   A and B reads dealt out evenly
  outer step (the next step is in the next slab)
     up to row block rb - ahead   the last A operands of this slab
     then                         my loads of the next slab have landed, my reads of this one
                                  too; barrier: so have everybody's
     the rest                     B and A operands of the next step, alternating with the
                                  request for the slabs of A and of B that go where this one's
                                  were (a group); what does not fit follows in the next step

An operand by rows is one ds_read_b128; turned over it is two ds_read_b64_tr_b16, each of which
gives sixteen lanes four k-values of their column from four rows of sixteen columns: twice the
reads, as many bytes, and no transposed copy of the operand in memory.  More reads behind the
barrier need it earlier, hence `ahead`.

Every memory operation gets an MFMA to itself.  All s_waitcnt are computed from the order of
issue (the counter holds 15: a wait for more becomes one for 14), and every operand is checked to
be the one that its MFMA expects.

Registers (v = VGPR, a = AGPR, s = SGPR):
  a[32i+4o : +3]      accumulator of row block i, operand o
  v[32b+4o : +3]      B operands, buffer b (step parity)
  v[64+4i : +3]       A operand of row block i
  v[96...] v[120...]  LDS addresses of the A and B reads: by rows 2 slot + step; turned over
                      8 slot + block
  v[144+t]            byte offsets of this lane's loads, A then B; of an operand by rows past
                      everything, by v160, for the last slab, where the lane's k-values are past the
                      end of the rows (turned over a slab ends with the window, rows do not)
  s[40:43] s[44:47]   buffer resources of A and B; the base moves on by a slab with every request
  s49 s50 s48 s51     slabs, requested of A and of B, left
  s52 s53 s60 s61     sizes of A and B for a slab, and for the last one (0 past it)
  s[54:56] s[57:59]   LDS addresses of this wave's part of the slots, A and B
  s62 s63             bytes from one slab to the next, A and B
"""
import math
import sys

RA, RB = 40, 44
S_REQB, S_N, S_REQA, S_LEFT, S_FULLA, S_FULLB, S_MA, S_MB = 48, 49, 50, 51, 52, 53, 54, 57
S_LASTA, S_LASTB, S_STEPA, S_STEPB = 60, 61, 62, 63
V_A, V_B, V_OFF, V_PAST = 96, 120, 144, 160
ROW = 128           # bytes of a row of 64 k-values
TURNED = 512        # bytes of a k-value's 256 columns
STEPS = 2           # of 32 k-values in a slab
LDS = 160 * 1024
TYPES = {"f16": "v_mfma_f32_16x16x32_f16", "bf16": "v_mfma_f32_16x16x32_bf16"}


class Shape:
    def __init__(self, layout, rb):
        self.layout, self.rb = layout, rb
        self.turn_a, self.turn_b = layout == "both", layout in ("b", "both")
        self.ahead = {"rows": 3, "b": 4, "both": 5}[layout]
        if self.ahead > rb - 1:
            self.ahead = rb - 1
        # load instructions per wave and slab, 1 KiB each (a turned A is always 256 columns wide)
        self.ta = 8 if self.turn_a else rb
        self.loads = self.ta + 8
        self.slab_a = 64 * TURNED if self.turn_a else 32 * rb * ROW
        self.slab_b = 256 * ROW
        # slabs of either operand in LDS
        self.ring_a = 3 if 3 * (self.slab_a + self.slab_b) <= LDS else 2
        self.ring_b = 3
        assert self.ring_a * self.slab_a + self.ring_b * self.slab_b <= LDS
        self.a_reads, self.b_reads = 1 + self.turn_a, 1 + self.turn_b
        room = 8 * self.ahead - 8 * self.b_reads - self.ahead * self.a_reads
        self.tail = min(self.loads, room)  # loads requested right behind the barrier
        assert self.tail > 0


def q(base): return f"v[{base}:{base + 3}]"
def d(base): return f"v[{base}:{base + 1}]"
def aq(base): return f"a[{base}:{base + 3}]"
def sq(base): return f"s[{base}:{base + 3}]"
def BOP(b, o): return 32 * b + 4 * o
def AOP(i): return 64 + 4 * i


class Emitter:
    def __init__(self):
        self.lines = []
        self.lds = []       # destinations of LDS reads in flight, oldest first
        self.vm = []        # slabs of the loads in flight, oldest first
        self.content = {}   # register quad -> what was last read into it
        self.aside = []     # blocks that the last requests branch to

    def emit(self, text):
        self.lines.append(text)

    def read(self, dst, text, tag):
        self.emit(text)
        self.lds.append(dst)
        self.content.setdefault(dst, [])
        if not self.content[dst] or self.content[dst][0] != tag:
            self.content[dst] = [tag, 0]
        self.content[dst][1] += 1

    def need(self, wants):
        """wait until the reads into these registers have landed (LDS reads land in order)"""
        for reg, tag, count in wants:
            assert self.content.get(reg) == [tag, count], (reg, tag, self.content.get(reg))
        regs = [reg for reg, _, _ in wants]
        last = max([i for i, r in enumerate(self.lds) if r in regs], default=-1)
        if last >= 0:
            left = min(len(self.lds) - last - 1, 14)
            self.lds = self.lds[len(self.lds) - left:]
            self.emit(f"s_waitcnt lgkmcnt({left})")


def request_head(e, sh, group):
    """what the loads of a group need, A of one slab and B of another: bases, m0, and aside, for the last
    slab of either operand and those past it, sizes and offsets"""
    n = len(e.aside)
    block = [f".Lff_last{n}_%=:"]
    operands = ((RA, S_REQA, S_LASTA, S_FULLA, S_STEPA, group + sh.ring_a, sh.turn_a, range(sh.ta), "a"),
                (RB, S_REQB, S_LASTB, S_FULLB, S_STEPB, group + sh.ring_b, sh.turn_b, range(sh.ta, sh.loads), "b"))
    for res, req, last, full, step, slab, turned, loads, name in operands:
        if slab < 0:
            continue
        if slab > 0:
            e.emit(f"s_add_u32 s{res}, s{res}, s{step}")
            e.emit(f"s_addc_u32 s{res + 1}, s{res + 1}, 0")
        e.emit(f"s_add_u32 s{req}, s{req}, 1")
        block += [f"s_cmp_eq_u32 s{req}, s{S_N}", f"s_cselect_b32 s{res + 2}, s{last}, s{full}",
                  f"s_cmp_le_u32 s{req}, s{S_N}", f"s_cselect_b32 s{res + 2}, s{res + 2}, 0"]
        if not turned:
            block += [f"s_cmp_lg_u32 s{req}, s{S_N}", f"s_cbranch_scc1 .Lff_not{n}{name}_%="]
            block += [f"v_or_b32 v{V_OFF + t}, v{V_OFF + t}, v{V_PAST}" for t in loads]
            block += [f".Lff_not{n}{name}_%=:"]
    # (of B at least as many slabs have been requested as of A)
    assert sh.ring_b >= sh.ring_a
    e.emit(f"s_cmp_ge_u32 s{S_REQB}, s{S_N}")
    e.emit(f"s_cbranch_scc1 .Lff_last{n}_%=")
    e.emit(f".Lff_back{n}_%=:")
    e.aside.append(block + [f"s_branch .Lff_back{n}_%="])
    if group + sh.ring_a >= 0:
        e.emit(f"s_mov_b32 m0, s{S_MA + (group + sh.ring_a) % sh.ring_a}")
    else:
        e.emit(f"s_mov_b32 m0, s{S_MB + (group + sh.ring_b) % sh.ring_b}")


def request(e, sh, group, t):
    """load t of a group, A's and then B's; m0 is left ready for load t + 1 (an MFMA or a nop lies
    between)"""
    of_a = t < sh.ta
    e.emit(f"buffer_load_dwordx4 v{V_OFF + t}, {sq(RA if of_a else RB)}, 0 offen lds")
    e.vm.append(group + (sh.ring_a if of_a else sh.ring_b))
    if t == sh.ta - 1:
        e.emit(f"s_mov_b32 m0, s{S_MB + (group + sh.ring_b) % sh.ring_b}")
    elif t < sh.loads - 1:
        e.emit("s_add_u32 m0, m0, 0x400")


def wait_for_slab(e, slab):
    """... to have landed (loads complete in order)"""
    last = max([i for i, at in enumerate(e.vm) if at <= slab], default=-1)
    e.vm = e.vm[last + 1:]
    assert len(e.vm) < 64
    return f"s_waitcnt vmcnt({len(e.vm)})"


def assign(ops, n):
    """(preferred MFMA, operation) -> {MFMA: operation}, distinct, in the order of preference"""
    at, last = {}, -1
    for pref, fn in sorted(ops, key=lambda x: x[0]):
        last = max(last + 1, int(pref))
        at[last] = fn
    assert last < n, last
    return at


def reads_of(turned, addr, dst, slot, h, block, tag):
    """the LDS reads of an operand, one or two functions"""
    if not turned:
        return [lambda e: e.read(dst, f"ds_read_b128 {q(dst)}, v{addr + 2 * slot + h} offset:{block * 16 * ROW}", tag)]
    return [lambda e, j=j: e.read(dst, f"ds_read_b64_tr_b16 {d(dst + 2 * j)}, v{addr + 8 * slot + block} "
                                       f"offset:{(32 * h + 4 * j) * TURNED}", tag) for j in range(2)]


# `at` is the step: slab 2 at, or 2 at + 1, and its half
def read_a(sh, at, i):
    return reads_of(sh.turn_a, V_A, AOP(i), at // 2 % sh.ring_a, at % 2, i, ("a", at, i))


def read_b(sh, at, o):
    return reads_of(sh.turn_b, V_B, BOP(at & 1, o), at // 2 % sh.ring_b, at % 2, o, ("b", at, o))


def next_operands(sh, at):
    """the reads of step `at` that the outer step before it issues, in order"""
    ops = read_b(sh, at, 0) + read_a(sh, at, 0)
    for o in range(1, 8):
        ops += read_b(sh, at, o)
    for i in range(1, sh.ahead):
        ops += read_a(sh, at, i)
    return ops


def step(e, sh, mfma, now, carry):
    """one step; carry: (group, first load) of a request that the step before left unfinished"""
    rb, ahead = sh.rb, sh.ahead
    ops = []
    for i in range(rb - ahead):
        ops += [(8 * i + x, fn) for x, fn in enumerate(read_a(sh, now, i + ahead))]
    for x, t in enumerate(range(carry[1], sh.loads) if carry else ()):
        ops.append((2 + 4 * x, lambda e, t=t: request(e, sh, carry[0], t)))
    left = None
    if now % STEPS == STEPS - 1:
        bar, slab = 8 * (rb - ahead), now // STEPS

        def barrier(e):
            e.emit(wait_for_slab(e, slab + 1) + " lgkmcnt(0)")
            e.lds = []
            e.emit("s_barrier")
            request_head(e, sh, slab)

        ops.append((bar - 1, barrier))
        behind = []
        reads = next_operands(sh, now + 1)
        loads = [lambda e, t=t: request(e, sh, slab, t) for t in range(sh.tail)]
        while reads or loads:  # in turns, and what is left of either
            if reads:
                behind.append(reads.pop(0))
            if loads:
                behind.append(loads.pop(0))
        ops += [(bar + x * 1e-3, fn) for x, fn in enumerate(behind)]
        left = (slab, sh.tail) if sh.tail < sh.loads else None
    else:
        for i in range(ahead):
            ops += [(8 * (rb - ahead + i) + x, fn) for x, fn in enumerate(read_a(sh, now + 1, i))]
        for o in range(8):
            ops += [(rb * o + 2 + x, fn) for x, fn in enumerate(read_b(sh, now + 1, o))]
    at = assign(ops, 8 * rb)
    b = now & 1
    for i in range(rb):
        for o in range(8):
            e.need([(AOP(i), ("a", now, i), sh.a_reads)] + ([(BOP(b, o), ("b", now, o), sh.b_reads)] if i == 0 else []))
            acc = 32 * i + 4 * o
            e.emit(f"{mfma} {aq(acc)}, {q(BOP(b, o))}, {q(AOP(i))}, {aq(acc)}")
            if 8 * i + o in at:
                at[8 * i + o](e)
    return left


def generate(sh, mfma):
    e = Emitter()
    # prologue: every slot requested (the last group as far as an outer step would have), the
    # accumulators zeroed, the first step's operands read
    e.emit(f"s_mov_b32 s{S_REQA}, 0")
    e.emit(f"s_mov_b32 s{S_REQB}, 0")
    e.emit(f"s_mov_b32 s{S_LEFT}, s{S_N}")
    for s in range(1, sh.ring_a):
        e.emit(f"s_add_u32 s{S_MA + s}, s{S_MA}, {s * sh.slab_a}")
    for s in range(1, sh.ring_b):
        e.emit(f"s_add_u32 s{S_MB + s}, s{S_MB}, {s * sh.slab_b}")
    for group in range(-max(sh.ring_a, sh.ring_b), 0):
        request_head(e, sh, group)
        for t in range(sh.loads if group < -1 else sh.tail):
            if group + (sh.ring_a if t < sh.ta else sh.ring_b) >= 0:
                e.emit("s_nop 0")
                request(e, sh, group, t)
    for n in range(32 * sh.rb):
        e.emit(f"v_accvgpr_write_b32 a{n}, 0")
    e.emit(wait_for_slab(e, 0))
    e.emit("s_barrier")
    for fn in next_operands(sh, 0):
        fn(e)
    carry = (-1, sh.tail) if sh.tail < sh.loads else None
    turn = math.lcm(sh.ring_a, sh.ring_b)  # slabs after which all slots come round

    def state():
        return ([(r, e.content[r]) for r in sorted(e.content)], list(e.lds), list(e.vm), carry)

    start = state()
    e.emit(".Lff_loop_%=:")
    for now in range(2 * turn):
        carry = step(e, sh, mfma, now, carry)
        if now % STEPS == STEPS - 1:
            e.emit(f"s_sub_u32 s{S_LEFT}, s{S_LEFT}, 1")
            e.emit(f"s_cmp_eq_u32 s{S_LEFT}, 0")
            e.emit("s_cbranch_scc0 .Lff_loop_%=" if now == 2 * turn - 1 else "s_cbranch_scc1 .Lff_done_%=")
    # the loop closes: what is in flight, and what is ready for the first step, is what it
    # started with, `turn` slabs on
    end = state()
    assert end[1] == start[1] and end[2] == [at + turn for at in start[2]]
    assert (end[3] and (end[3][0] - turn, end[3][1])) == start[3]
    ready = [(r, [(c[0][0], c[0][1] - 2 * turn, c[0][2]), c[1]]) for r, c in end[0] if c[0][1] == 2 * turn]
    assert ready == [(r, c) for r, c in start[0] if c[0][1] == 0]
    e.emit(".Lff_done_%=:")
    # the last MFMAs' results are not readable for 18 cycles, and the hardware does not
    # interlock that for what follows; nothing may be on its way into LDS or registers either
    e.emit("s_nop 15")
    e.emit("s_nop 15")
    e.emit("s_waitcnt vmcnt(0) lgkmcnt(0)")
    e.emit("s_branch .Lff_end_%=")
    for block in e.aside:
        e.lines += block
    e.emit(".Lff_end_%=:")
    return e.lines


def statement(sh, mfma):
    out = ["// generated by gen_products.py -- do not edit", "asm volatile("]
    out += [f'    "{l}\\n\\t"' for l in generate(sh, mfma)]
    outs = [f'"={{{aq(32 * i + 4 * o)}}}"(acc[{i}][{o}])' for i in range(sh.rb) for o in range(8)]
    outs += [f'"+{{{sq(RA)}}}"(ra_words)', f'"+{{{sq(RB)}}}"(rb_words)']
    by_rows = [t for t in range(sh.loads) if not (sh.turn_a if t < sh.ta else sh.turn_b)]
    outs += [f'"+{{v{V_OFF + t}}}"(src[{t}])' for t in by_rows]
    out.append("    : " + ",\n      ".join(outs))
    ins = [f'"{{s{S_N}}}"(slabs)', f'"{{s{S_MA}}}"(lds_a)', f'"{{s{S_MB}}}"(lds_b)',
           f'"{{s{S_FULLA}}}"(full_a)', f'"{{s{S_FULLB}}}"(full_b)', f'"{{s{S_LASTA}}}"(last_a)',
           f'"{{s{S_LASTB}}}"(last_b)', f'"{{s{S_STEPA}}}"(step_a)', f'"{{s{S_STEPB}}}"(step_b)']
    ins += [f'"{{v{V_A + j}}}"(a_rd[{j}])' for j in range((8 if sh.turn_a else 2) * sh.ring_a)]
    ins += [f'"{{v{V_B + j}}}"(b_rd[{j}])' for j in range((8 if sh.turn_b else 2) * sh.ring_b)]
    ins += [f'"{{v{V_OFF + t}}}"(src[{t}])' for t in range(sh.loads) if t not in by_rows]
    if by_rows:
        ins.append(f'"{{v{V_PAST}}}"(past)')
    out.append("    : " + ",\n      ".join(ins))
    clob = [f"v{n}" for n in range(64 + 4 * sh.rb)]
    clob += [f"s{S_REQA}", f"s{S_REQB}", f"s{S_LEFT}"]
    clob += [f"s{S_MA + s}" for s in range(1, sh.ring_a)] + [f"s{S_MB + s}" for s in range(1, sh.ring_b)]
    clob += ["scc", "memory"]  # (m0 is the compiler's to reserve; it keeps nothing there)
    out.append("    : " + ", ".join(f'"{c}"' for c in clob) + ");")
    return "\n".join(out) + "\n"


if __name__ == "__main__":
    outdir = sys.argv[1] if len(sys.argv) > 1 else "."
    for type, mfma in TYPES.items():
        for layout in ("rows", "b", "both"):
            for rb in (5, 6, 7, 8):
                with open(f"{outdir}/ff_{type}_{layout}_{rb}.inc", "w") as f:
                    f.write(statement(Shape(layout, rb), mfma))
