"""No kernel of the built operator library spills registers to memory: the metadata of every kernel in it names a private segment of
zero bytes and no spilled vector registers."""
import re

from elixir_amd import _ops_abi


def integer(data, at):
    """A MessagePack integer."""
    b = data[at]
    if b < 0x80:
        return b
    size = {0xCC: 1, 0xCD: 2, 0xCE: 4, 0xCF: 8}[b]
    return int.from_bytes(data[at + 1:at + 1 + size], 'big')


def test_no_kernel_spills_registers():
    with open(_ops_abi.LIB_PATH, 'rb') as f:
        data = f.read()
    kernels = 0
    for m in re.finditer(rb'\.private_segment_fixed_size', data):
        end = data.index(rb'.wavefront_size', m.start())
        record = data[m.start():end]
        name = re.search(rb'(_ZN[\w]*?)\.kd', record).group(1).decode()
        values = {key: integer(record, record.index(key) + len(key)) for key in (b'.private_segment_fixed_size', b'.vgpr_spill_count')}
        assert not any(values.values()), (name, values)
        kernels += 1
    assert kernels > 300    # the metadata was there to be read
