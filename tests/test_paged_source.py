"""What can be seen in the paged cache's kernels without running them."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'motif_b200', 'csrc')


def kernels():
    """(name, parameters, body) of every kernel of the paged cache."""
    for path in sorted(glob.glob(os.path.join(CSRC, 'kv4*.cu'))):
        text = re.sub(r'//[^\n]*', '', open(path).read())
        for m in re.finditer(r'__global__[^;{]*?(\w+_kernel)\(([^{;]*)\)\s*\{', text):
            yield m.group(1), m.group(2), text[m.end():text.index('\n}\n', m.end())]


@pytest.mark.parametrize('name,parameters,body', list(kernels()), ids=lambda v: v if str(v).endswith('_kernel') else '')
def test_kernels_wait_before_they_touch_memory(name, parameters, body):
    """They start while the kernel before them in the stream ends, and only its end (griddepcontrol.wait)
    makes what it and the ones before it wrote visible."""
    assert 'wait_for_previous()' in body
    before = body[:body.index('wait_for_previous()')]
    pointers = [re.findall(r'\w+', p)[-1] for p in parameters.split(',') if '*' in p]
    members = re.findall(r'\*\s*(\w+)|\*(\w+),', re.search(r'struct Args \{(.*?)\n\};', open(os.path.join(
        CSRC, 'kv4_attention.cu')).read(), re.S).group(1))
    used = [p for p in pointers if re.search(rf'\b{p}\b', before)]
    used += [m for pair in members for m in pair if m and re.search(rf'\ba\.{m}\b', before)]
    used += re.findall(r'\b(?:scan_requests|locate|advance|tiles_of|length_of|queries_of|store4|load8)\b', before)
    assert not used, f'{name} reads or writes before it waits: {used}'


def test_every_kernel_is_found():
    assert [k[0] for k in kernels()] == ['paged_reserve_kernel', 'paged_release_kernel', 'kv4_append_kernel',
                                         'kv4_gather_kernel', 'kv4_attention_kernel', 'kv4_merge_kernel']
