"""What ``check_spills`` finds in a listing of the training operators' kernels."""

from tileccl_amd.csrc import check_spills


def listing(name, spilled, body=("s_endpgm",)):
    return "\n".join([f"{name}:                ; @{name}", *("\t" + line for line in body), ".Lfunc_end0:", f"  - .name:           {name}", "    .sgpr_count:     32",
                      "    .vgpr_count:     128", f"    .vgpr_spill_count: {spilled}"]) + "\n"


def test_scratch_inside_the_weight_gradients_loop_counts():
    name = "_ZN4tccl22weight_gradient_kernelIDF16bfLi256ELi256ELb1ELi1EEEvNS_10WeightArgsE"
    asm = listing(name, 1, ("v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]", "scratch_load_dword v9, off, off",
                            "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]", "s_endpgm"))
    assert list(check_spills.kernels(asm)) == [(name, 128, 1, 1)]


def test_norm_kernels_that_keep_registers_in_scratch_are_listed():
    backward = "_ZN4tccl22layer_norm_grad_kernelI{}Li{}ELi{}ELb1ELi0ELb0EEEvNS_12NormGradArgsE"
    forward = "_ZN4tccl17layer_norm_kernelI{}Li{}ELi{}ELb0ELi0EEEvNS_8NormArgsE"
    cases = [(backward.format("DF16b", 4, 4), 85, True), (backward.format("DF16_", 4, 2), 2, True), (backward.format("DF16b", 8, 1), 6, True),
             (backward.format("DF16b", 8, 1), 40, False), (backward.format("f", 1, 1), 1, False), (forward.format("f", 1, 4), 16, True),
             (forward.format("DF16_", 2, 1), 3, False), (forward.format("DF16_", 2, 1), 0, None), ("_ZN4tccl11hold_kernelIDF16bLi1EEEvNS_8HoldArgsE", 5, None)]
    for name, spilled, known in cases:
        assert list(check_spills.norm_spills(listing(name, spilled))) == ([] if known is None else [(name, spilled, known)])
        assert check_spills.report(listing(name, spilled), 2) == (known is not False)
