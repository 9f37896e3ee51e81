"""CPU: the masked attention kernels exchange partials by the sequence that test_exchange_isa.py checks in the emitted assembly."""

import re

import pytest

from test_exchange_isa import check_exchange, device_assembly, is_partial_load, is_partial_store, kernel_body

KERNELS = ["_ZN3bpt17masked_few_kernelILi1ELi1ELb1ELb0ELb1EE", "_ZN3bpt17masked_few_kernelILi1ELi1ELb0ELb1ELb0EE",
           "_ZN3bpt18masked_many_kernelILi1ELi1ELb1ELb0ELi2EE", "_ZN3bpt18masked_many_kernelILi1ELi1ELb0ELb1ELi1EE"]


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    return device_assembly("masked_fp8_head.hip", tmp_path_factory.mktemp("isa"))


@pytest.mark.parametrize("prefix", KERNELS)
def test_partial_exchange_sequence(prefix, assembly):
    body = kernel_body(assembly, prefix)
    assert any(line.startswith("global_atomic_add") and re.search(r"\bsc0\b", line) for line in body), "no returning fetch-add"
    assert any(is_partial_store(line) for line in body) and any(is_partial_load(line) for line in body)
    problems = check_exchange(body)
    assert not problems, problems[:5]
