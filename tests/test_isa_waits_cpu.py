"""CPU checks of wait states in our own gfx950 build that the compiler does not place around inline assembly (the
CDNA ISA's table of manually inserted wait states; the compiler keeps both for its own instructions)."""
import re

import pytest

import test_isa_cpu as isa

pytestmark = isa.pytestmark


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    return isa.disassemble(isa.CODE_OBJECT, tmp_path_factory.mktemp("waits"))


def predecessors(ins):
    """Of each instruction of a kernel, those that may run right before it."""
    index, base = {a: i for i, (a, *_) in enumerate(ins)}, ins[0][0]
    before = [[] for _ in ins]
    for i, (_, m, _, target) in enumerate(ins):
        if m not in ("s_branch", "s_endpgm") and i + 1 < len(ins):
            before[i + 1].append(i)
        if target is not None and base + target[1] in index:
            before[index[base + target[1]]].append(i)
    return before


def too_early(ins, before, i, least, writes):
    """The last instruction for which `writes` holds with fewer than `least` wait states between it and instruction i."""
    todo = [(p, 0) for p in before[i]]
    while todo:
        at, waited = todo.pop()
        mnemonic, operands = ins[at][1:3]
        if writes(mnemonic, operands):
            return ins[at]
        waited += isa._waits(mnemonic, operands)
        if waited < least:
            todo += [(p, waited) for p in before[at]]
    return None


def loads_to_lds(mnemonic, operands):
    return mnemonic.startswith("global_load_lds") or mnemonic.startswith("buffer_load") and re.search(r"\blds\b", operands)


def test_a_load_to_lds_waits_for_m0(kernels):
    """A scalar write of M0, one wait state, a load to LDS, which takes its place there from M0."""
    seen, flagged = 0, []
    for name, ins in kernels.items():
        before = predecessors(ins)
        for i, (address, mnemonic, operands, _) in enumerate(ins):
            if loads_to_lds(mnemonic, operands):
                seen += 1
                at = too_early(ins, before, i, 1, lambda m, ops: m.startswith("s_") and ops.split(",")[0].strip() == "m0")
                if at is not None:
                    flagged.append(f"{name}+{address - ins[0][0]:#x}: {mnemonic} behind {at[1]} {at[2]}")
    assert seen > 1000
    assert not flagged, f"{len(flagged)}: " + "\n".join(flagged[:20])


def scalar_registers(token):
    m = re.match(r"s\[(\d+):(\d+)\]$", token) or re.match(r"s(\d+)()$", token)
    return set(range(int(m.group(1)), int(m.group(2) or m.group(1)) + 1)) if m else set()


def scalars_of_valu(mnemonic, operands):
    """Scalar registers that a vector instruction writes."""
    if not mnemonic.startswith("v_"):
        return set()
    tokens = isa._operands(operands)
    carry = tokens[1:2] if "_co_" in mnemonic or mnemonic.startswith("v_mad_u64") or mnemonic.startswith("v_div_scale") else []
    return set().union(*(scalar_registers(t) for t in tokens[:1] + carry))


def test_memory_instructions_wait_for_scalars_that_vector_instructions_wrote(kernels):
    """A vector instruction's write of a scalar register (v_readfirstlane), five wait states, a vector memory
    instruction that reads it: before, the register may hold an older address."""
    seen, flagged = 0, []
    for name, ins in kernels.items():
        before = predecessors(ins)
        for i, (address, mnemonic, operands, _) in enumerate(ins):
            if not mnemonic.startswith(("global_", "buffer_", "flat_", "scratch_")):
                continue
            read = set().union(*(scalar_registers(t) for t in re.split(r",\s*|\s+", operands)))
            if read:
                seen += 1
                at = too_early(ins, before, i, 5, lambda m, ops: read & scalars_of_valu(m, ops))
                if at is not None:
                    flagged.append(f"{name}+{address - ins[0][0]:#x}: {mnemonic} {operands} behind {at[1]} {at[2]}")
    assert seen > 1000
    assert not flagged, f"{len(flagged)}: " + "\n".join(flagged[:20])


def test_data_of_wide_stores_is_not_written_before_it_is_read(kernels):
    """A store of more than 8 bytes a lane reads its data registers late: a vector instruction may write them two wait
    states after it."""
    seen, flagged = 0, []
    for name, ins in kernels.items():
        before = predecessors(ins)
        for i, (address, mnemonic, operands, _) in enumerate(ins):
            tokens = isa._operands(operands)
            written = isa._regs(tokens[0]) if mnemonic.startswith("v_") and tokens else set()

            def stores(m, ops):
                if not re.match(r"(global|flat|scratch|buffer)_store_dwordx[34]$", m):
                    return False
                return isa._regs(isa._operands(ops)[0 if m.startswith("buffer") else 1].split()[0]) & written
            if written:
                seen += 1
                at = too_early(ins, before, i, 2, stores)
                if at is not None:
                    flagged.append(f"{name}+{address - ins[0][0]:#x}: {mnemonic} {operands} behind {at[1]} {at[2]}")
    assert seen > 1000
    assert not flagged, f"{len(flagged)}: " + "\n".join(flagged[:20])


def test_mfma_results_are_not_read_early_on_any_way(kernels):
    """The wait states from each matrix instruction to the first vector read of its result, on every way through any
    number of branches, are at least the fewest that the compiler places inside a block."""
    needed, flagged = {}, []
    for ins in kernels.values():
        for i, (_, mnemonic, operands, _) in enumerate(ins):
            if not mnemonic.startswith("v_mfma"):
                continue
            result, waited = isa._regs(isa._operands(operands)[0]), 0
            for _, m, ops, target in ins[i + 1:i + 40]:
                if target is not None or m == "s_endpgm":
                    break
                if result & isa._reads(m, ops):
                    needed[mnemonic] = min(needed.get(mnemonic, 99), waited)
                    break
                if m.startswith("v_mfma") and result & isa._regs(isa._operands(ops)[0]):
                    break
                waited += isa._waits(m, ops)
    assert needed
    for name, ins in kernels.items():
        before = predecessors(ins)
        for i, (address, mnemonic, operands, _) in enumerate(ins):
            reads = isa._reads(mnemonic, operands)
            todo, seen = [(p, 0) for p in before[i]] if reads else [], set()
            while todo:
                at, waited = todo.pop()
                m, ops = ins[at][1:3]
                written = isa._regs(isa._operands(ops)[0]) if m.startswith("v_") else set()
                if m.startswith("v_mfma") and reads & written:
                    if waited < needed.get(m, 8):
                        flagged.append(f"{name}+{address - ins[0][0]:#x}: {mnemonic} {operands} {waited} < {needed.get(m, 8)} behind {m}")
                    continue
                waited += isa._waits(m, ops)
                if waited < 20 and not reads <= written and (at, waited) not in seen:
                    seen.add((at, waited))
                    todo += [(p, waited) for p in before[at]]
    assert not flagged, f"{len(flagged)}, of {needed}: " + "\n".join(flagged[:20])
