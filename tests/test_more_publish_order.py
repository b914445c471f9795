"""The order of stores, wait, barrier and count of the decode over 8-bit caches and of
the decode behind shared keys, in the emitted code, as test_isa_publish_order.py has
it for the other kernels whose workgroups leave parts for the last one."""
from test_isa_publish_order import CSRC, arrival, check_publish_order, device_asm, functions


def test_decode_over_8_bits_publishes_before_counting(tmp_path):
    asm = device_asm(CSRC / "attn_decode_q8.hip", tmp_path)
    found = [(n, b) for n, b in functions(asm) if "decode_q8_kernel" in n]
    assert len(found) == 3 * 3 * 2  # head sizes, query heads at once, formats
    for name, body in found:
        check_publish_order(name, arrival(body))  # every thread stores, one counts


def test_decode_behind_shared_keys_publishes_before_counting(tmp_path):
    asm = device_asm(CSRC / "attn_decode_own.hip", tmp_path)
    found = [(n, b) for n, b in functions(asm) if "decode_batch_kernel" in n]
    assert len(found) == 4 * 4  # head sizes, query heads at once
    for name, body in found:
        check_publish_order(name, arrival(body))
