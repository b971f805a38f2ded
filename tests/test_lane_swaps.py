"""The device code of the library as built: a vector register that lanes exchange (v_permlane16_swap, v_permlane32_swap) or that
another lane reads (a DPP operand) was written at least two wait states before, along every path.  The hardware does not wait for it;
the compiler keeps the distance behind its own instructions, but does not see one that stands in a block of assembly."""
from test_device_code import _registers, kernels, listings  # noqa: F401  (a fixture)


def early_exchanges(listing):
    """(kernel, wait states, the instruction that writes, the one that exchanges) of every pair that is too close."""
    for name, code, after in kernels(listing, "v_"):
        if not any(o.startswith("v_permlane") or "_dpp" in o for o, _, _ in code):
            continue
        for i, (op, args, _) in enumerate(code):
            if not op.startswith("v_") or op.startswith(("v_mfma", "v_cmp", "v_readlane", "v_readfirstlane", "v_nop")):
                continue
            both = op.startswith(("v_permlane16_swap", "v_permlane32_swap", "v_swap"))    # these write their second operand as well
            result, todo = _registers(",".join(args.split(",")[:2 if both else 1])), [(j, 0) for j in after(i)]
            while todo:
                j, waited = todo.pop()
                if j is None or j >= len(code) or waited >= 2:
                    continue
                o, a, _ = code[j]
                operands = a.split(",")
                moved = operands[:2] if o.startswith("v_permlane") else operands[1:2] if "_dpp" in o else []
                if result & _registers(",".join(moved)):
                    yield name, waited, f"{op} {args}", f"{o} {a}"
                    continue
                todo += [(k, waited + (int(a, 0) + 1 if o == "s_nop" else 1)) for k in after(j)]


def test_exchanged_registers_were_written_two_states_before(listings):  # noqa: F811
    code = ["v_mov_b32_e32 v7, v3", "s_nop 1", "s_nop 0", "v_permlane16_swap_b32_e32 v3, v7", "v_mov_b32_dpp v8, v7 row_mirror row_mask:0xf bank_mask:0xf",
            "v_add_f32_e32 v9, v8, v8", "s_endpgm"]

    def found(order):
        return len([*early_exchanges("0000 <k>:\n" + "".join(f"\t{code[i]} // {4 * n:08X}: 0\n" for n, i in enumerate(order)))])
    assert found((0, 1, 3, 6)) == found((2, 0, 1, 4, 6)) == found((0, 2, 5, 3, 6)) == 0
    assert found((0, 3, 6)) == found((0, 2, 3, 6)) == found((0, 2, 4, 6)) == found((1, 0, 5, 4, 6)) == 1
    assert sum(t.count("_swap_b32") for t, _ in listings) > 100            # the listings are what they should be
    assert not [v for t, _ in listings for v in early_exchanges(t)][:5]


def test_exchanges_are_between_two_registers(listings):  # noqa: F811
    """A swap of a register with itself is what the copies in front of them are there against."""
    found = [(name, a) for t, _ in listings for name, code, _ in kernels(t, "v_permlane")
             for o, a, _ in code if o.startswith(("v_permlane16_swap", "v_permlane32_swap"))]
    assert len(found) > 100 and not [f for f in found if len(_registers(f[1])) != 2][:5]
