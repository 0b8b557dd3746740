// Prints what the GGUF reader makes of a file's rotary scaling: kind, factor, trained, beta_fast, beta_slow, then the frequency
// factors.  A std::runtime_error is printed as "ERROR <message>" with exit code 3.
#include <cstdio>

#include "../../litenn_b200/host/GGUFReader.hpp"

int main(int argc, char** argv)
{
	if (argc != 2)
	{
		return 2;
	}
	try
	{
		LiteNN::B200::GGUF::Archive archive(argv[1]);
		const auto r = archive.ParseRopeScaling();
		std::printf("%d %.9g %.9g %.9g %.9g", r.scaling.kind, r.scaling.factor, r.scaling.trained, r.scaling.beta_fast, r.scaling.beta_slow);
		for (const float f : r.frequencyFactors)
		{
			std::printf(" %.9g", f);
		}
		std::printf("\n");
		return 0;
	}
	catch (const std::runtime_error& e)
	{
		std::printf("ERROR %s\n", e.what());
		return 3;
	}
}
