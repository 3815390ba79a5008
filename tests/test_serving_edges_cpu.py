"""Refusals of the serving operators at the ends of their ranges: arguments are checked before anything touches a device."""
from test_serving_cpu import HERE, attention, refused, rules


def test_rules_refuse_vocabularies_that_steps_over_them_would_leave():
    # a step of 16384 tokens from the last multiple below 2^31 ends beyond 32 bits
    refused(rules(vocab=2 ** 31 - 1, ld_logits=2 ** 31, ld_out=2 ** 31), "dimensions")
    refused(rules(vocab=2 ** 30 + 1, ld_logits=2 ** 31, ld_out=2 ** 31), "dimensions")


def test_attention_refuses_its_queries_as_output_and_scales_that_overflow():
    # every block reads its rows while others may have written theirs
    refused(attention(d_out=HERE), "output")
    # 2.36e38 * log2(e) is the largest fp32 number
    refused(attention(scale=2.4e38, d_out=HERE + 4096), "scale")
