"""Names of what leaves a code in the fault word: host side only."""
import pytest


@pytest.mark.parametrize("codes,word", [((1, 4, 12, 24, 35), "FFN"), ((40, 47, 55), "barrier"), ((61, 64), "product"),
                                        ((71, 75), "weight gradient"), ((81, 82), "Adam"), ((0,), "no kernel"),
                                        ((56, 99, -3), "kernel")])
def test_origin_of_a_code(codes, word):
    from mole_b200 import ops
    for code in codes:
        assert word in ops.device_fault_origin(code)


def test_status_carries_the_message_of_its_own_thread():
    from mole_b200 import _lib
    _lib.check(0)
    with pytest.raises(_lib.MoleError, match="MOLE_ERR_DEVICE: said elsewhere") as e:
        _lib.check(-6, "said elsewhere")
    assert e.value.status == -6
