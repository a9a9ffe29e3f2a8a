"""The build's limits on scratch memory (noeira_amd/build.py): the first entry that a kernel's name holds counts, kernels
without one are not looked at, and every entry names a kernel of its source."""
import os
import re

from noeira_amd import build as B

REMARKS = "".join(f"""a.hip:1:1: remark: Function Name: _ZN2nq12_GLOBAL__N_1{name} [-Rpass-analysis=kernel-resource-usage]
a.hip:1:1: remark:     VGPRs: 128 [-Rpass-analysis=kernel-resource-usage]
a.hip:1:1: remark:     ScratchSize [bytes/lane]: {n} [-Rpass-analysis=kernel-resource-usage]
""" for name, n in (("22layer_norm_grad_kernelILi1024ELi2ELb1ELb1ELb1EE", 84), ("22layer_norm_grad_kernelILi1024ELi2ELb0ELb1ELb1EE", 88),
                    ("22layer_norm_grad_kernelILi512ELi1ELb1ELb1ELb1EE", 4), ("17layer_norm_kernelILi1024ELi2ELb0ELb0EE", 28),
                    ("17layer_norm_kernelILi1024ELi2ELb1ELb0EE", 28), ("26layer_norm_grad_sum_kernelE", 0), ("11zero_kernelE", 64)))


def test_kernels_beyond_their_limit_are_named():
    got = B._beyond_scratch(REMARKS, B.SCRATCH_LIMITS["nq_norm.hip"])
    assert [(k.split("N_1")[1][2:], n) for k, n in got] == [
        ("layer_norm_grad_kernelILi1024ELi2ELb0ELb1ELb1EE", 88), ("layer_norm_grad_kernelILi512ELi1ELb1ELb1ELb1EE", 4),
        ("layer_norm_kernelILi1024ELi2ELb1ELb0EE", 28)]
    assert B._beyond_scratch(REMARKS, ()) == [] and B._beyond_scratch("", B.SCRATCH_LIMITS["nq_norm.hip"]) == []


def test_limited_kernels_exist_where_they_are_listed():
    for src, limits in B.SCRATCH_LIMITS.items():
        text = open(os.path.join(B.CSRC, src)).read()
        for part, _ in limits:
            name = re.match(r"[a-z_]+?_(?=kernelI|$)", part).group(0)
            assert re.search(rf"void {name}\w*kernel\(", text), (src, part)
